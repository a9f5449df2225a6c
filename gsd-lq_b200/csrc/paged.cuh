// paged.cuh -- what the kernels over a paged cache share: the rows of a call, and the host's checks.
#pragma once
#include "common.cuh"

namespace gsdlq {

// Positions above it are refused, so that a row's length rounded up to whole tiles stays within an int, whatever the
// table allows.
constexpr int PAGED_MAX_POS = INT32_MAX - 128;

// Sequence of row r, and how many positions it has with its own (0: idle).  `flag`: report what is wrong
// with it (once per launch is enough).
struct PagedRow {
  int seq, len;
};
__device__ __forceinline__ PagedRow paged_row(const gsdlq_paged_kv_t& kv, const int* row_seq, const int* pos, int r,
                                              bool flag) {
  const int p = pos[r], s = row_seq ? row_seq[r] : r;
  if (p == -1) return {s, 0};
  if (s < 0 || s >= kv.n_seqs) {
    if (flag) raise_flag(GSDLQ_FLAG_BAD_PAGE);
    return {s, 0};
  }
  if (p < 0 || p > PAGED_MAX_POS || (long long)p >= (long long)kv.max_blocks * kv.page_size) {
    if (flag) raise_flag(GSDLQ_FLAG_BAD_POS);
    return {s, 0};
  }
  return {s, p + 1};
}

__device__ __forceinline__ bool paged_valid(const gsdlq_paged_kv_t& kv, int page) {
  return page >= 0 && page < kv.n_pages;
}

// ---- host checks
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool pages_ok(const gsdlq_paged_kv_t& kv) {  // table and counts
  return kv.table && kv.refs && kv.n_pages > 0 && kv.n_pages <= (1 << 28) && kv.page_size > 0 && kv.max_blocks > 0 && kv.n_seqs > 0 &&
         kv.n_seqs <= GSDLQ_PAGED_MAX_SEQS;
}
inline bool pool_ok(const gsdlq_paged_kv_t& kv) {  // and the pool itself
  return pages_ok(kv) && kv.k && kv.v && aligned16(kv.k) && aligned16(kv.v) && kv.layers > 0 && kv.n_kv_heads > 0 &&
         (kv.kv_type == GSDLQ_KV_F16 || kv.kv_type == GSDLQ_KV_BF16) &&
         (kv.head_dim == 32 || kv.head_dim == 64 || kv.head_dim == 128);
}
inline bool rows_ok(const gsdlq_paged_kv_t& kv, const int* row_seq, const int* pos, int rows) {
  return pos && rows > 0 && (row_seq || rows <= kv.n_seqs);
}

}  // namespace gsdlq
