// What the kernels over the paged 8-bit cache share: its layout, and how they
// read the numbers that only the device knows (lengths, row ranges, page
// numbers), none of which is trusted with an address.
#pragma once

#include "mx_common.h"

namespace mx {
namespace kv8 {

#define KV8_HD __host__ __device__ __forceinline__

// The most tokens that a row of the page table may hold: token numbers, a tile past the
// last among them, are ints.
constexpr long long kMostTokens = 1LL << 30;

// Tokens of a sequence in the cache: kv_lens[b], at least 0 and at most what its
// row of the page table can hold.
KV8_HD int cut_len(int len, int max_pages, int lp) {
  const long long most = (long long)max_pages << lp;
  return len < 0 ? 0 : (long long)len > most ? (int)most : len;
}

// The rows first .. last-1 of sequence b: cu[b] .. cu[b+1], cut to 0 .. T and never
// negative in number.
struct Rows {
  int first, last;
};
KV8_HD Rows cut_rows(int from, int to, int T) {
  from = from < 0 ? 0 : from > T ? T : from;
  to = to < from ? from : to > T ? T : to;
  return Rows{from, to};
}
KV8_HD Rows rows_of(const int* cu, int b, int T) {
  return cu ? cut_rows(cu[b], cu[b + 1], T) : cut_rows(b, b + 1, T);
}

// The page that holds token t, or -1: past the table's row, or a number that is no
// page of the pool.
KV8_HD int page_of(const int* row, int t, int lp, int max_pages, int pages) {
  const int j = t >> lp;
  if (t < 0 || j >= max_pages) return -1;
  const int p = row[j];
  return p >= 0 && p < pages ? p : -1;
}

inline int log2_page(int page) { return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : page == 128 ? 7 : -1; }

// The sizes that every entry point checks the same way.
inline int check_cache(const void* k, const void* v, const void* ks, const void* vs, int n_kv, int d, int page,
                       int pages) {
  if (!k || !v || !ks || !vs) return MX_ERR_NULL;
  if (n_kv <= 0 || pages <= 0 || (d != 64 && d != 128) || log2_page(page) < 0) return MX_ERR_SHAPE;
  if ((long long)pages * n_kv > 0x7fffffffLL) return MX_ERR_SHAPE;
  if (((uintptr_t)k | (uintptr_t)v) & 15) return MX_ERR_ALIGN;
  if (((uintptr_t)ks | (uintptr_t)vs) & 3) return MX_ERR_ALIGN;
  return MX_OK;
}

}  // namespace kv8
}  // namespace mx
