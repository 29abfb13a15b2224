// Attention over a cache: what the kernels and the host share.  Keys and values lie in pages that a block table names,
// or one after the other; a sequence's new tokens are its last ones; a window hides all but the last keys and the sinks.
#pragma once
#include <cstdint>
#include <cuda.h>

#include "common.cuh"

namespace ma {

struct CacheArgs {
  const uint16_t* q;
  uint16_t* o;
  float* lse;
  int32_t* status;
  long long qs[3], os[3];  // element strides: sequence, head, token (ragged: the first is 0)
  long long ls[2];         // of lse: sequence, head
  const int* table;        // [B][table_width] page numbers; null: keys of sequence b lie in "page" b, one after the other
  long long table_stride;
  const int* seq_lens;     // [B] tokens of each sequence, the new ones among them; null: Nk
  const int* cu_q;         // [B + 1] first row of each sequence in q; null: Nq rows each
  long long diag;          // without seq_lens: query token i sees keys up to diag + i
  int B, Hq, Hkv, G, D;
  int Nq, Nk, total_q;
  int page_shift, n_pages, table_width;  // page size 1 << page_shift
  int window, sinks;       // window 0: none
  int key0;                // keys before it are another launch's (a shared prefix)
  float scale_log2;
  FastDiv by_g, by_nq;
  // fwd_cache_ws.cu: query heads that share a Q tile (all G of a KV head, or 1), tokens of each in it, pairs of Q tiles of a
  // sequence (not ragged), groups of `pack` heads, tiles that a piece of an item has at least
  int pack, tpt, pairs, groups, min_tiles;
  int pair_items;          // not ragged: CTAs before this one take two Q tiles, those from it on one each
  int cut;                 // ragged: items are cut so that all together make about this many pieces (0: not)
  FastDiv by_pack, by_pairs, by_groups, by_gqa;
  int shared;              // a launch over a shared prefix: its tokens
  // scratch: pieces of cut items, un-normalised
  float* part_o;
  float2* part_ml;         // (row maximum in log2 units, row sum)
  int* counters;           // zero between launches
  // Not null: nothing is written to o; every row's un-normalised O and (m, l) go here, [rows of q * Hq][D] and
  // [rows of q * Hq], for the launch that adds the shared prefix's pieces.
  float* rest_o;
  float2* rest_ml;
};

// x / y, neither negative.  Not inlined on the device: a kernel's start is bound by the code it fetches for the first time.
#ifdef __CUDACC__
static __host__ __device__ __noinline__ long long cache_div(long long x, long long y) {
#else
inline long long cache_div(long long x, long long y) {
#endif
  if (((x | y) >> 31) == 0) return static_cast<uint32_t>(x) / static_cast<uint32_t>(y);
  return x / y;
}

// One sequence of a call.  Keys that some row of it sees: [lo, hi) and, with a window, [0, sink_end) before them.
struct CacheSeq {
  long long row0;   // first row in q of a ragged call (0 otherwise: the stride of the sequence says where)
  long long diag;   // query token i sees keys up to diag + i
  int nq, lo, hi, sink_end;
  bool bad;         // a length or a row number outside the call's tensors
};

__host__ __device__ inline int clamp_to(long long x, long long lo, long long hi) {
  return static_cast<int>(x < lo ? lo : x > hi ? hi : x);
}

__host__ __device__ inline CacheSeq cache_seq(const CacheArgs& a, int first_row, int end_row, int seq_len) {
  CacheSeq s;
  s.bad = false;
  if (a.cu_q != nullptr) {
    const int r0 = clamp_to(first_row, 0, a.total_q), r1 = clamp_to(end_row, r0, a.total_q);
    s.bad = r0 != first_row || r1 != end_row;
    s.row0 = r0;
    s.nq = r1 - r0;
  } else {
    s.row0 = 0;
    s.nq = a.Nq;
  }
  long long len = a.Nk;
  s.diag = a.diag;
  if (a.seq_lens != nullptr) {
    const long long room = static_cast<long long>(a.table_width) << a.page_shift;
    len = clamp_to(seq_len, 0, room < 0x7fffff00ll ? room : 0x7fffff00ll);  // rounded up to tiles it fits in 31 bits
    s.bad = s.bad || len != seq_len;
    s.diag = len - s.nq;
  }
  s.hi = clamp_to(s.diag + s.nq, 0, len);
  s.lo = a.key0;
  if (a.window > 0) s.lo = clamp_to(s.diag + 1 - a.window, s.lo, 0x7fffffff);
  if (s.lo > s.hi) s.lo = s.hi;
  s.sink_end = a.window > 0 ? (a.sinks < s.lo ? a.sinks : s.lo) : 0;
  return s;
}

// Keys [*first, *end) that query token i of a sequence sees, and of those before them the first a.sinks.
__host__ __device__ inline void cache_row(const CacheArgs& a, const CacheSeq& s, int i, int* first, int* end) {
  *end = clamp_to(s.diag + i + 1, 0, s.hi);
  *first = a.key0;
  if (a.window > 0) *first = clamp_to(s.diag + i + 1 - a.window, a.key0, 0x7fffffff);
}

// Tiles of kTile keys that hold the keys [lo, hi) and [0, sink_end): number j of them is tile j up to n_sink, and
// first + (j - n_sink) from there on.  At least one, so that every row is written.
struct CacheTiles {
  int n_sink, first, n;
  __host__ __device__ int at(int j) const { return j < n_sink ? j : first + (j - n_sink); }
};
template <int kTile>
__host__ __device__ inline CacheTiles cache_tiles(int lo, int hi, int sink_end) {
  CacheTiles t;
  t.n_sink = (sink_end + kTile - 1) / kTile;
  t.first = lo / kTile;
  if (t.first < t.n_sink) t.first = t.n_sink;
  const int end = (hi + (kTile - 1)) / kTile;
  t.n = t.n_sink + (end > t.first ? end - t.first : 0);
  if (t.n < 1) t.n = 1;
  return t;
}

// Whether [k, k + n) holds keys that no row sees.
__host__ __device__ inline bool cache_partly_seen(int lo, int hi, int sink_end, int k, int n) {
  return k + n > hi || (k < lo && sink_end < lo && k + n > sink_end);
}

// Whether some row sees one of the keys [k, k + n).
__host__ __device__ inline bool cache_seen(int lo, int hi, int sink_end, int k, int n) {
  return k < hi && ((k + n > lo && lo < hi) || k < sink_end);
}

}  // namespace ma
