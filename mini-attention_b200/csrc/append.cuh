// Appending new tokens to a paged cache: what the kernel and the host share.
#pragma once
#include <cstdint>

#include "common.cuh"

namespace ma {

struct AppendArgs {
  const uint16_t *k, *v, *q;       // new tokens; q may be null
  uint16_t *k_cache, *v_cache, *q_out;
  long long ks[3], vs[3], qs[3], qos[3];  // element strides: sequence, head, token (ragged: the first is 0)
  long long kcs[3], vcs[3];        // element strides of the caches: page, head, token of the page
  const float* rope;               // [rope_rows][rot]: cosines of the rot / 2 angles of a position, then their sines; or null
  const int* table;                // [B][table_width] page numbers
  const int* seq_lens;             // [B] tokens of each sequence, the new ones among them
  const int* cu_q;                 // [B + 1] first row of each sequence; null: n rows each
  int32_t* status;
  long long table_stride;
  int B, n, rows, Hq, Hkv, D;
  int rot, interleaved, rope_rows;
  int page_shift, n_pages, table_width;
  FastDiv by_n, by_units;
};

// Whether a sequence of a ragged call lies outside its tensors, also one that no row of the call belongs to.
__host__ __device__ inline bool append_outside(const AppendArgs& a, int first_row, int end_row, int seq_len) {
  return first_row < 0 || end_row < first_row || end_row > a.rows || seq_len < 0 ||
         seq_len > static_cast<long long>(a.table_width) << a.page_shift;
}

// Where row t of a sequence goes.
struct AppendSlot {
  bool none;            // the row belongs to no sequence: it is left as it is, and so is its query
  bool held;            // the cache has a place for it (not for one before the sequence's first token)
  bool bad;             // a length, a row, a page or a position outside the call's tensors
  int pos;
  long long page;       // page and token of the page, where held
  int at;
};
// `first`: the sequence's first row, `n_new`: its rows.  The block table is looked up by the caller's function.
template <typename Table>
__host__ __device__ inline AppendSlot append_slot(const AppendArgs& a, int t, long long first, long long n_new, int seq_len,
                                                  const Table& table) {
  AppendSlot s{};
  const bool rows_bad = first < 0 || first + n_new > a.rows || t >= first + n_new;  // the last where row numbers fall
  if (t < first || rows_bad) {  // before the first sequence's rows
    s.none = true;
    s.bad = rows_bad;
    return s;
  }
  const long long pos = seq_len - n_new + (t - first);
  const long long room = static_cast<long long>(a.table_width) << a.page_shift;
  if (pos < 0) {  // the front of a padded sequence
    s.bad = seq_len < 0;
    return s;
  }
  if (pos >= room || (a.rope != nullptr && pos >= a.rope_rows)) {
    s.bad = true;
    return s;
  }
  s.pos = static_cast<int>(pos);
  const int page = table(s.pos >> a.page_shift);
  if (page < 0 || page >= a.n_pages) {
    s.bad = true;
    return s;
  }
  s.held = true;
  s.page = page;
  s.at = s.pos & ((1 << a.page_shift) - 1);
  return s;
}

}  // namespace ma
