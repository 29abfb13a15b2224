// Attention over a cache for many query rows per KV head (chunked prefill, a prefix that a batch shares, prefill with a
// sliding window): the mathematics of fwd_cache.cu on tcgen05, in the division of labour of fwd_ws.cu.
//
//   item      = two 128-row Q tiles of one sequence and one KV head; the `pack` query heads of the KV head share them, row r of
//               a tile is token r / pack, head r % pack
//   warps 0-3 softmax of Q tile 0 (thread = row), its epilogue; warps 4-7 the same for Q tile 1
//   warp 8    MMA issuer of Q tile 0, warp 10 of Q tile 1
//   warp 9    finds the item, copies Q and K; warp 11 copies V (and zeroes padding rows of the Q tiles before that)
//
// An item visits the 128-key tiles that its rows see: those of the sinks, then those from the window of its first row to its
// last row's position, each as two 64-key halves.  Where there are few items their tiles are cut into pieces: every piece
// leaves (un-normalised O, m, l) in scratch and counts itself in, and the one that counts in last folds them, in their order.
//
// Tiles at the ends hold keys that no row of the sequence sees and that may be anything.  Their scores are replaced; their
// rows of V are cleared in shared memory by warp 11, which hands such a tile over itself instead of leaving that to the copy.
//
// Bound: tensor pipe and power where items are long (16384 tokens, 32/8 heads of 128, window 4096, 4 sinks 878 us = 1.1 PFLOP/s;
// 1.7 us a 128-key step of a CTA at the power cap).  Short windows are bound by a CTA's ends and by the tiles that only some of
// its 256 rows see: 4 x 1024 tokens, 12 heads of 64, window 256 20.6 us, 3 us of an item's 12 outside its steps.
//
// Few items: their pairs are taken apart, a Q tile to a CTA; a CTA's step then takes 0.8 of a pair's and there is nothing to
// fold (rules and figures: cache_plan in api.cu, ragged_item).
//
// The query heads of a KV head always share Q tiles: a pair of tiles then spans 256 / G tokens, and its band of keys is that
// much narrower.
//
// Built and dropped: one CTA an SM that walks a contiguous part of all items' tiles (cut evenly, no second wave).  Its start
// takes 4.5 us instead of 1.5, and without the offset that each item gives its second Q tile the two softmax groups fall into
// step, in which a 64-key half takes 1750 clk instead of 1520: both calls above took 14 % longer, only mixed chunks gained.  Turns
// that keep the groups apart, through a barrier between the MMA warps, cost more than the step (2000 clk).  Two CTAs of one Q tile
// each on an SM (D = 64, four ring slots, half of TMEM): as quick as single tiles on SMs of their own where those fit, and 4096
// tokens, 12 heads, window 1024 took 106 us instead of 98.7, 1024 tokens, window 256 the same: the groups fall into step.
#include <atomic>

#include "cache.cuh"
#include "launch.cuh"
#include "ptx.cuh"

namespace ma {

namespace {

constexpr int kThreads = 384;
constexpr int kWarpMma0 = 8, kWarpTma = 9, kWarpMma1 = 10, kWarpV = 11;
constexpr int kHalfN = kTileN / 2;   // keys per half tile
constexpr float kSumLimit = 256.0f;  // a half's sum of P above which the row's reference moves
// registers per thread after setmaxnreg: 8 * 208 + 4 * 88 = 12 * 168, what the launch allocates
constexpr int kRegSoftmax = 208;
constexpr int kRegOther = 88;

template <int D>
struct Layout {
  static constexpr int kBoxes = D / kBoxCols;
  static constexpr int kTileBytes = kBoxes * kBoxBytes;  // Q, K or V tile (32 KB at D = 128)
  static constexpr int kStages = (D == 128) ? 4 : 8;     // ring slots, each one K or V tile
  static constexpr int kOffQ = 0;                        // two Q tiles (reused as O staging)
  static constexpr int kOffRing = 2 * kTileBytes;
  static constexpr int kOffBar = kOffRing + kStages * kTileBytes;
  // barrier indices (8 bytes each); [t][h] = index + 2 * t + h
  static constexpr int kBarQFull = 0;                       // [2]
  static constexpr int kBarKvFull = 2;                      // [kStages]
  static constexpr int kBarKvEmpty = kBarKvFull + kStages;  // [kStages]
  static constexpr int kBarSFull = kBarKvEmpty + kStages;   // [2][2] MMA -> softmax
  static constexpr int kBarPReady = kBarSFull + 4;          // [2][2] softmax -> MMA
  static constexpr int kBarODone = kBarPReady + 4;          // [2][2] MMA -> softmax (rescale, epilogue)
  static constexpr int kBarStagger = kBarODone + 4;         // one-shot: tile 0 published its first row maxima
  static constexpr int kBarRaw = kBarStagger + 1;           // copy of a V tile that warp 11 hands over itself
  static constexpr int kNumBars = kBarRaw + 1;
  static constexpr int kOffMisc = kOffBar + kNumBars * 8;   // tmem slot, abort flag, arrival order [2]
  static constexpr int kOffItem = kOffMisc + 32;            // WsItem
  static constexpr int kBytes = kOffItem + 96;
  static constexpr int kDynSmem = kBytes + 1024;
  static constexpr int kTmemCols = 512;
  static constexpr int kColS = 0;    // S buffer of (tile t, half h) at kColS + 128 * t + 64 * h
  static constexpr int kColO = 256;  // O accumulator of tile t at kColO + D * t
};

// What a CTA works on: found by the producer warp, read by the others.
struct WsItem {
  CacheSeq s;
  CacheTiles t;
  int b, q0, nt, group;     // sequence, first query token, Q tiles that hold rows (0: no item), group of heads
  int j0, n;                // tiles [j0, j0 + n) of t
  int part, n_parts, slot0; // piece of the item, pieces in all, slot of scratch of the first
};
static_assert(sizeof(WsItem) <= 96, "WsItem");

__device__ __forceinline__ float part_weight(float m, float mt) { return m == -INFINITY ? 0.f : ex2(m - mt); }
__device__ __forceinline__ float row_lse(float m, float l) {
  return l == 0.f ? -INFINITY : m * 0.6931471805599453f + __logf(l);
}
// bits [0, x) of 64
__device__ __forceinline__ uint64_t below(int x) { return x <= 0 ? 0ull : x >= 64 ? ~0ull : (1ull << x) - 1; }

// What a lane copies of a 128-key tile: 64 columns of the keys of one page.  Pages are fetched a tile ahead, since the ring has
// no room for the time that takes.
template <int kBoxes>
struct PageLane {
  int shift, sub, bx;  // keys of a box (1 << shift: a page's, at most 128), the lane's among the tile's, its columns
  int page = 0, key = 0, next_page = 0, next_key = 0;
  bool wanted = false, next_wanted = false;
  __device__ __forceinline__ PageLane(const CacheArgs& a)
      : shift(a.table != nullptr ? min(7, a.page_shift) : 7), sub((threadIdx.x & 31) / kBoxes), bx((threadIdx.x & 31) % kBoxes) {}
  __device__ __forceinline__ void fetch(const CacheArgs& a, const WsItem& it, int j) {  // tile number j of the item
    next_key = it.t.at(j) * kTileN + (sub << shift);
    next_wanted = sub < (kTileN >> shift) && cache_seen(it.s.lo, it.s.hi, it.s.sink_end, next_key, 1 << shift);
    next_page = it.b;
    if (a.table != nullptr && next_wanted) next_page = a.table[it.b * a.table_stride + (next_key >> a.page_shift)];
  }
  __device__ __forceinline__ void settle(const CacheArgs& a) {
    page = next_page;
    key = next_key;
    wanted = next_wanted;
    if (a.table != nullptr) {
      key &= (1 << a.page_shift) - 1;
      if (wanted && static_cast<unsigned>(page) >= static_cast<unsigned>(a.n_pages)) {
        wanted = false;
        if (a.status != nullptr) atomicOr(a.status, kErrCache);
      }
    }
  }
  __device__ __forceinline__ void copy(const CUtensorMap* tm, uint32_t dst, uint32_t full, int hk) const {  // the whole warp
    const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, wanted)) * (128u << shift);
    if ((threadIdx.x & 31) == 0) mbar_expect_tx(full, bytes);
    __syncwarp();
    if (wanted) tma_load_4d(dst + bx * kBoxBytes + ((sub << shift) << 7), tm, full, bx * kBoxCols, key, hk, page);
    __syncwarp();
  }
};

// Give-up path: copies may still be in flight; let them land (bounded) before the shared memory is released.
__device__ __forceinline__ void wait_for_copies() {
  const uint64_t t0 = global_timer_ns();
  while (global_timer_ns() - t0 < 2000000ull) {
  }
}

// Which piece of which item CTA x of a ragged launch works on; the whole warp.  False: none.  Lengths are known here only, so
// every CTA adds up the tiles of all sequences: pieces are at most half as long as an SM's share, and where the sequences are
// few those with the most keys come first.  (One piece per pair, sequences in their order: 148 SMs wait for the last of 192
// items of 100 tiles, 357 us where all items together are 237 on each SM.)  Where single Q tiles fill no more than a CTA per SM
// and no piece of a pair would be much shorter than they are, each is an item (*single: which of its pair).
__device__ __forceinline__ bool ragged_item(const CacheArgs& a, int x, WsItem* it, int* pair, int* single) {
  const int lane = threadIdx.x & 31;
  int span = 2 * a.tpt;
  auto look = [&](int b, CacheSeq* s, int* pairs, int* tiles) {
    *pairs = 0;
    *tiles = 1;
    if (b >= a.B) return;
    *s = cache_seq(a, a.cu_q[b], a.cu_q[b + 1], a.seq_lens[b]);
    *pairs = (s->nq + (span - 1)) / span;
    long long seen = s->hi;
    if (a.window > 0) seen = min(seen, static_cast<long long>(a.window) + span + a.sinks + kTileN);
    *tiles = max(1, static_cast<int>((seen + (kTileN - 1)) / kTileN));
  };
  CacheSeq s{};
  int pairs, tiles, most = 0x7fffffff;  // tiles of a piece
  // Sequences out of range are reported by the first CTA for all, since those left without rows are nobody's item.  Here and not
  // in the pass below: kept there, `bad` took mixed chunks of 342 us to 348; 40 short sequences gained 0.2 us of 18.9.
  if (x == 0 && a.status != nullptr) {
    bool bad = false;
    for (int b = lane; b < a.B; b += 32) bad |= cache_seq(a, a.cu_q[b], a.cu_q[b + 1], a.seq_lens[b]).bad;
    if (bad) atomicOr(a.status, kErrCache);
  }
  if (a.cut > 0) {
    long long total = 0, items = 0, apart = 0;
    int longest = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
      look(b0 + lane, &s, &pairs, &tiles);
      total += static_cast<long long>(pairs) * tiles;
      items += pairs;
      if (pairs > 0) {
        apart += (s.nq + (a.tpt - 1)) / a.tpt;
        longest = max(longest, tiles);
      }
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      total += __shfl_xor_sync(0xffffffffu, total, d);
      items += __shfl_xor_sync(0xffffffffu, items, d);
      apart += __shfl_xor_sync(0xffffffffu, apart, d);
    }
    longest = __reduce_max_sync(0xffffffffu, longest);
    const long long even = (total * a.groups + a.cut - 1) / a.cut;
    // Rows that overlap, which only row numbers that fall give, may be more than the launch has CTAs for: a piece without one
    // would leave its item's counter standing, so nothing is cut then.
    if (items * a.groups + a.cut <= gridDim.x) most = clamp_to(even, 2 * a.min_tiles, 0x7fffffff);
    // 2 x 128 tokens against 1600 keys, 32/8 heads of 128: 21.6 us, 26.2 in pieces of pairs; 300 against 2040, 8/2 heads 24.0
    // and 27.0.  Not where most pairs are single tiles as it is (3 x 100 tokens, 12 heads: 24.9, 23.1 in pieces).
    if (2 * apart * a.groups <= a.cut && 2 * apart >= 3 * items && longest <= max(most, 4 * a.min_tiles)) {
      span = a.tpt;
      most = 0x7fffffff;
    }
  }
  long long before = 0;  // pieces of the sequences before
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    look(b0 + lane, &s, &pairs, &tiles);
    const int parts = (tiles - 1) / most + 1;
    const long long count = static_cast<long long>(pairs) * a.groups * parts;
    long long first = before, all = 0;
    for (int o = 0; o < 32; ++o) {
      const long long c = __shfl_sync(0xffffffffu, count, o);
      const int t = __shfl_sync(0xffffffffu, tiles, o);
      if (t > tiles || (t == tiles && o < lane)) first += c;
      all += c;
    }
    const uint32_t mine = __ballot_sync(0xffffffffu, x >= first && x < first + count);
    if (mine != 0) {
      const int l = __ffs(mine) - 1;
      it->b = b0 + l;
      const int at = static_cast<int>(x - __shfl_sync(0xffffffffu, first, l));
      it->n_parts = __shfl_sync(0xffffffffu, parts, l);
      const int idx = at / it->n_parts;
      it->part = at - idx * it->n_parts;
      const int back = div_by(idx, a.by_groups);
      it->group = idx - back * a.groups;
      *pair = __shfl_sync(0xffffffffu, pairs, l) - 1 - back;  // the latest first: it sees the most keys
      if (span == a.tpt) {
        *single = *pair & 1;
        *pair >>= 1;
      }
      it->s = cache_seq(a, a.cu_q[it->b], a.cu_q[it->b + 1], a.seq_lens[it->b]);
      return true;
    }
    before += all;
  }
  return false;
}

}  // namespace

// PREFIX: the rows are those of all sequences, one after the other, the keys the a.shared first tokens of them; every piece is
// left for cache_merge_kernel, nothing is written to o.
// NARROW: head dim 96 on the D = 128 tiles, the MMAs leave the 32 columns of zeros out.
template <int D, bool BF16, bool PREFIX, bool NARROW>
__global__ void __launch_bounds__(kThreads, 1)
fwd_cache_ws_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                    const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_o, const CacheArgs a) {
  using L = Layout<D>;
  constexpr int kCols = NARROW ? 96 : D;  // head dim the MMAs work on
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t sbase = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (sbase - raw);

  const uint32_t sQ = sbase + L::kOffQ;
  const uint32_t sRing = sbase + L::kOffRing;
  const uint32_t bars = sbase + L::kOffBar;
  auto bar = [&](int idx) -> uint32_t { return bars + 8u * idx; };
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gbase + L::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gbase + L::kOffMisc + 8);
  volatile int* arrival = reinterpret_cast<volatile int*>(gbase + L::kOffMisc + 16);  // [2 tiles]
  WsItem* item_s = reinterpret_cast<WsItem*>(gbase + L::kOffItem);

  grid_dep_launch();
  const int tid = threadIdx.x;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // warp-uniform for the compiler
  const int lane = tid & 31;
  const int tpt = a.tpt;
  const WaitCtx wc{abort_flag, a.status, MINIATTN_WAIT_LIMIT_NS};

  PageLane<L::kBoxes> pl(a);  // warps 9 and 11

  if (warp == kWarpTma) {
    for (int i = lane; i < L::kNumBars; i += 32) {
      uint32_t count = 1;  // Q full, K/V full, raw, S full, O done: one arrival (a copy, an MMA commit)
      if (i >= L::kBarKvEmpty && i < L::kBarSFull) count = 2;      // one release per Q tile (see below where there is one)
      else if (i >= L::kBarPReady && i < L::kBarODone) count = 4;  // P ready: 4 warps
      else if (i == L::kBarStagger) count = 4;                     // the 4 softmax warps of tile 0, once
      mbar_init(bar(i), count);
    }
    if (lane == 0) {
      *abort_flag = 0;
      prefetch_tmap(&tm_q);
      prefetch_tmap(&tm_k);
      prefetch_tmap(&tm_v);
    }
    fence_mbar_init();
    fence_proxy_async_smem();
    __syncwarp();
    grid_dep_wait();

    WsItem it{};
    int x = static_cast<int>(blockIdx.x), pair, single = -1;
    bool there = true;
    if (PREFIX || a.cu_q == nullptr) {
      if (x >= a.pair_items) {  // the last wave's pairs, a Q tile to a CTA
        single = (x - a.pair_items) & 1;
        x = a.pair_items + ((x - a.pair_items) >> 1);
      }
      const int idx = div_by(x, a.by_groups);
      it.group = x - idx * a.groups;
      it.b = PREFIX ? 0 : div_by(idx, a.by_pairs);
      pair = a.pairs - 1 - (idx - it.b * a.pairs);
      it.part = static_cast<int>(blockIdx.y);
      it.n_parts = static_cast<int>(gridDim.y);
      it.slot0 = x * static_cast<int>(gridDim.y);
      if constexpr (PREFIX) {
        it.s.nq = a.cu_q != nullptr ? a.total_q : a.B * a.Nq;
        // Read through the block table of the longest sequence: others may be padding, or end before the prefix does.  Only a
        // sequence that has rows and whose rows and length are in range: nobody needs the pages of the others.
        const auto usable = [&](int b) {
          const CacheSeq s = cache_seq(a, a.cu_q != nullptr ? a.cu_q[b] : 0, a.cu_q != nullptr ? a.cu_q[b + 1] : 0, a.seq_lens[b]);
          return s.nq > 0 && !s.bad;
        };
        int longest = -1;
        for (int b = lane; b < a.B; b += 32)
          if (usable(b)) longest = max(longest, a.seq_lens[b]);
        longest = __reduce_max_sync(0xffffffffu, longest);
        int of = a.B - 1;
        for (int b = lane; b < a.B; b += 32)
          if (a.seq_lens[b] == longest && usable(b)) of = min(of, b);
        it.b = __reduce_min_sync(0xffffffffu, of);
        it.s.hi = clamp_to(min(a.shared, longest), 0, static_cast<long long>(a.table_width) << a.page_shift);
      } else {
        it.s = cache_seq(a, 0, 0, a.seq_lens != nullptr ? a.seq_lens[it.b] : 0);
      }
    } else {
      there = ragged_item(a, x, &it, &pair, &single);
      it.slot0 = x - it.part;
    }
    if (there) {
      if (it.s.bad && lane == 0 && a.status != nullptr) atomicOr(a.status, kErrCache);
      it.q0 = (pair * 2 + (single > 0 ? 1 : 0)) * tpt;
      it.nt = it.q0 >= it.s.nq ? 0 : single < 0 && it.q0 + tpt < it.s.nq ? 2 : 1;
      // keys that rows of these tiles see
      int lo = it.s.lo, hi = it.s.hi, sink_end = it.s.sink_end;
      if constexpr (!PREFIX) {
        int first, end;
        cache_row(a, it.s, it.q0, &lo, &end);
        cache_row(a, it.s, max(min(it.q0 + it.nt * tpt, it.s.nq) - 1, 0), &first, &hi);
        lo = min(max(lo, it.s.lo), hi);
        sink_end = a.window > 0 ? min(a.sinks, lo) : 0;
      }
      it.t = cache_tiles<kTileN>(lo, hi, sink_end);
      if (lo >= hi && sink_end == 0) it.t.n = 0;
      if (!PREFIX) it.n_parts = max(1, min(it.n_parts, it.t.n / a.min_tiles));  // a prefix's pieces are all added up
      if (it.part >= it.n_parts) {
        it.nt = 0;
      } else {
        it.j0 = static_cast<int>(static_cast<long long>(it.t.n) * it.part / it.n_parts);
        it.n = static_cast<int>(static_cast<long long>(it.t.n) * (it.part + 1) / it.n_parts) - it.j0;
      }
    }
    if (lane == 0) *item_s = it;
    if (it.nt > 0 && it.n > 0) {
      // The first copies start here, before TMEM is allocated and the CTA synchronises.
      if (lane == 0) {
        for (int t = 0; t < it.nt; ++t) {
          // a box holds tpt tokens of pack heads, heads fastest: rows [0, pack * tpt) of the tile
          mbar_expect_tx(bar(L::kBarQFull + t), L::kBoxes * a.pack * tpt * 128);
          for (int bx = 0; bx < L::kBoxes; ++bx)
            tma_load_5d(sQ + t * L::kTileBytes + bx * kBoxBytes, &tm_q, bar(L::kBarQFull + t), bx * kBoxCols, 0,
                        static_cast<int>(it.s.row0) + it.q0 + t * tpt, it.group, PREFIX || a.cu_q != nullptr ? 0 : it.b);
        }
      }
      __syncwarp();
      pl.fetch(a, it, it.j0);
      pl.settle(a);
      if (it.n > 1) pl.fetch(a, it, it.j0 + 1);
      pl.copy(&tm_k, sRing, bar(L::kBarKvFull), div_by(it.group, a.by_gqa));
    }
  }
  if (warp == kWarpMma0) {
    tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), L::kTmemCols);
    tmem_relinquish();
  }
  {
    // where pack does not divide 128 the last rows of the Q tiles belong to nobody; zeros keep their scores finite
    const int pad = kTileM - a.pack * tpt;
    if (warp == kWarpV && pad > 0) {
      for (int i = lane; i < 2 * L::kBoxes * pad * 8; i += 32) {
        const int box = i / (pad * 8), at = i % (pad * 8);
        *reinterpret_cast<uint4*>(gbase + L::kOffQ + box * kBoxBytes + (kTileM - pad) * 128 + at * 16) =
            make_uint4(0u, 0u, 0u, 0u);
      }
      fence_proxy_async_smem();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  grid_dep_wait();  // every thread: they read lengths and write results
  const WsItem it = *item_s;
  const int nt = it.nt, n_tiles = it.n;

  if (warp < 8) {
    // =========================== softmax ===========================================
    reg_inc<kRegSoftmax>();
    const int t = warp >> 2;
    if (t < nt) {
      const int r = tid & 127;
      const int in_tile = div_by(r, a.by_pack);
      const int tok = it.q0 + t * tpt + in_tile;                // query token of this thread
      const int head = it.group * a.pack + (r - in_tile * a.pack);
      const bool real = tok < it.s.nq && in_tile < tpt;
      const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t tS = tmem_base + L::kColS + 128 * t + lane_off;
      const uint32_t tO = tmem_base + L::kColO + D * t + lane_off;
      const float c = a.scale_log2;
      // the keys that this row sees
      int first, end;
      if constexpr (PREFIX) {
        first = 0;
        end = it.s.hi;
        if (real) {
          int b, i, r0 = 0, r1 = 0;
          if (a.cu_q != nullptr) {
            int lo = 0, hi = a.B;  // the last sequence whose first row is not behind this one
            while (lo < hi) {
              const int mid = (lo + hi + 1) >> 1;
              if (a.cu_q[mid] <= tok) lo = mid;
              else hi = mid - 1;
            }
            b = lo;
            if (b < a.B) {
              r0 = a.cu_q[b];
              r1 = a.cu_q[b + 1];
            }
            i = tok - r0;
          } else {
            b = div_by(tok, a.by_nq);
            i = tok - b * a.Nq;
          }
          if (b < a.B) {
            const CacheSeq s = cache_seq(a, r0, r1, a.seq_lens[b]);
            cache_row(a, s, i, &first, &end);
            end = min(end, it.s.hi);
          }
        }
        __syncwarp();
      } else {
        // rows that are nobody's see what their tile's last one does
        cache_row(a, it.s, min(it.q0 + t * tpt + min(in_tile, tpt - 1), it.s.nq - 1), &first, &end);
      }
      // what all rows of the warp see, so that the tiles in between need no look at their keys
      const int all_from = __reduce_max_sync(0xffffffffu, first), all_to = __reduce_min_sync(0xffffffffu, end);
      float m_cur = -INFINITY;  // running (lazily updated) row maximum, log2 units
      float l_run = 0.f;

      constexpr int kHalvesUnrolled = D == 128 ? 1 : 2;
      for (int j = 0; j < n_tiles; ++j) {
        const int k_tile = it.t.at(it.j0 + j) * kTileN;
#pragma unroll (kHalvesUnrolled)
        for (int hb = 0; hb < 2; ++hb) {
          mbar_wait(bar(L::kBarSFull + 2 * t + hb), j & 1, wc, kErrWaitS);
          tc_fence_after();
          uint32_t s[2][32];
          tmem_ld32(tS + hb * kHalfN, s[0]);
          tmem_ld32(tS + hb * kHalfN + 32, s[1]);
          tmem_wait_ld();
          const int k0 = k_tile + hb * kHalfN;
          bool sees = true;  // this row, some key of this half
          if (k0 < all_from || k0 + kHalfN > all_to) {
            // by selection: what a hidden key's score holds does not matter
            const uint64_t seen = below(end - k0) & (~below(first - k0) | below(a.sinks - k0));
            const uint32_t part[2] = {static_cast<uint32_t>(seen), static_cast<uint32_t>(seen >> 32)};
            sees = seen != 0;
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!((part[q] >> i) & 1u)) s[q][i] = __float_as_uint(-INFINITY);
          }
          // No row maximum is searched for in the usual half: the exponentials are taken against the reference the row
          // has, and their sum says whether it still serves (fwd_ws.cu).
          const bool start = (j == 0 && hb == 0);
          float psum0, psum1;
          uint32_t pk[32];
          bool fix = start;
          for (int pass = 0;; ++pass) {
            if (fix) {
              float mx4[4];
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                mx4[q] = -INFINITY;
#pragma unroll
                for (int i = 0; i < 16; i += 2)
                  mx4[q] = fmax3_nan(mx4[q], __uint_as_float(s[q >> 1][(q & 1) * 16 + i]),
                                     __uint_as_float(s[q >> 1][(q & 1) * 16 + i + 1]));
              }
              float mx = fmax3_nan(fmax3_nan(mx4[0], mx4[1], mx4[2]), mx4[3], mx4[3]) * c;  // log2 units, like m_cur
              if (!(mx < INFINITY)) mx = __int_as_float(0x7fffffff);  // a NaN or +inf makes the row's result a NaN
              float alpha = 1.f;
              if (!(mx <= m_cur)) {
                alpha = ex2(m_cur - mx);
                m_cur = mx;
              }
              if (!start && __any_sync(0xffffffffu, alpha != 1.f)) {
                l_run *= alpha;
                // every PV issued so far into O_t must have finished: the previous half-step's
                if (hb == 0) mbar_wait(bar(L::kBarODone + 2 * t + 1), (j - 1) & 1, wc, kErrWaitO);
                else mbar_wait(bar(L::kBarODone + 2 * t + 0), j & 1, wc, kErrWaitO);
                tc_fence_after();
#pragma unroll 1
                for (int q = 0; q < kCols / 32; ++q) {
                  uint32_t o[32];
                  tmem_ld32(tO + q * 32, o);
                  tmem_wait_ld();
#pragma unroll
                  for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                  tmem_st32(tO + q * 32, o);
                }
                tmem_wait_st();
              }
              if (t == 0 && start && pass == 0) warp_arrive(bar(L::kBarStagger));  // once
            }
            const float mc = (m_cur == -INFINITY) ? 0.f : m_cur;
            // A share of the exponentials by a polynomial on the FMA pipe, as in fwd_ws.cu; the quartic at every head dim:
            // rows that see a key or two show the cubic's 5e-5 in their lse.
            auto on_fma_pipe = [](int i) { return D == 64 ? (i & 7) == 0 : (i == 0 || i == 10 || i == 20); };
            uint64_t psum = pack_f32x2(0.f, 0.f);
            const uint64_t c2 = pack_f32x2(c, c), mc2 = pack_f32x2(-mc, -mc);
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                float x0, x1;
                unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(s[q][i]), __uint_as_float(s[q][i + 1])), c2, mc2), x0, x1);
                float p0, p1;
                if (on_fma_pipe(i)) {
                  exp2_poly_f32x2<true>(x0, x1, p0, p1);
                } else {
                  p0 = ex2(x0);
                  p1 = ex2(x1);
                }
                psum = add_f32x2(psum, pack_f32x2(p0, p1));
                // P in 16 bits for the second product: off by half a step of the type for each weight
                pk[q * 16 + (i >> 1)] = pack2<BF16>(p0, p1);
              }
            unpack_f32x2(psum, psum0, psum1);
            // again where the sum is too large, or the row sees its first keys
            if (pass == 1 || !__any_sync(0xffffffffu, !(psum0 + psum1 <= kSumLimit) || (m_cur == -INFINITY && sees))) break;
            fix = true;
          }
          l_run += psum0 + psum1;
          tmem_st32(tS + hb * kHalfN, pk);  // P of this half over the first 32 columns of its S
          tmem_wait_st();
          tc_fence_before();
          warp_arrive(bar(L::kBarPReady + 2 * t + hb));
        }
      }
      if (n_tiles > 0) {
        mbar_wait(bar(L::kBarODone + 2 * t + 1), (n_tiles - 1) & 1, wc, kErrWaitO);
        tc_fence_after();
      }
      // A row that saw no key keeps -inf; its hidden scores left 2^-126 terms in l_run (the polynomial holds its argument).  So
      // does a row that saw a NaN and in its last half nothing, whose sum stays the NaN it is.
      if (m_cur == -INFINITY && l_run == l_run) l_run = 0.f;
      auto chunk = [&](int q, uint32_t (&o)[32]) {  // 32 columns of this row's accumulator
        if (n_tiles > 0) {
          tmem_ld32(tO + q * 32, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
      };
      bool write_out = !PREFIX;
      float m_tot = m_cur, l_tot = l_run;
      // slots of the item's pieces: [piece][tile][D / 4][128 rows][4] floats, a warp stores 512 bytes in a row
      const long long slot0 = static_cast<long long>(it.slot0) * 2 + t;
      if (PREFIX || it.n_parts > 1) {
        const long long my = (slot0 + 2 * it.part) * kTileM;
        a.part_ml[my + r] = make_float2(m_cur, l_run);
        float4* po = reinterpret_cast<float4*>(a.part_o + my * D) + r;
#pragma unroll 1
        for (int q = 0; q < kCols / 32; ++q) {
          uint32_t o[32];
          chunk(q, o);
#pragma unroll
          for (int g = 0; g < 8; ++g)
            po[(q * 8 + g) * kTileM] = make_float4(__uint_as_float(o[4 * g]), __uint_as_float(o[4 * g + 1]),
                                                   __uint_as_float(o[4 * g + 2]), __uint_as_float(o[4 * g + 3]));
        }
      }
      if (!PREFIX && it.n_parts > 1) {
        __threadfence();  // release: the piece before the count
        named_bar_sync(1 + t, 128);
        if (r == 0) {
          __threadfence();
          int* cnt = a.counters + 2 * it.slot0 + t;
          const int order = atomicAdd(cnt, 1);
          if (order == it.n_parts - 1) *cnt = 0;
          arrival[t] = order;
        }
        named_bar_sync(1 + t, 128);
        write_out = arrival[t] == it.n_parts - 1;
        if (write_out) {
          __threadfence();  // acquire: every other piece was published before it was counted
          m_tot = -INFINITY;
          for (int p = 0; p < it.n_parts; ++p) m_tot = fmaxf(m_tot, __ldcg(a.part_ml + (slot0 + 2 * p) * kTileM + r).x);
          l_tot = 0.f;
          for (int p = 0; p < it.n_parts; ++p) {
            const float2 ml = __ldcg(a.part_ml + (slot0 + 2 * p) * kTileM + r);
            l_tot = fmaf(ml.y, part_weight(ml.x, m_tot), l_tot);
          }
        }
      }
      if (write_out) {
        // ---- O / l -> 16 bit -> swizzled smem (the tile's Q buffer) -> global memory ----
        if (real && a.lse != nullptr)
          a.lse[it.b * a.ls[0] + head * a.ls[1] + it.s.row0 + tok] =
              l_tot == 0.f ? -INFINITY : m_tot * 0.6931471805599453f + __logf(l_tot);
        __syncwarp();
        const float f = l_tot > 0.f ? 1.f / l_tot : l_tot;  // a NaN stays one
        const uint32_t stage = sQ + t * L::kTileBytes;
        // A warp's 32 rows of a box leave by TMA where they are whole tokens of this sequence; the last tokens of a ragged
        // one, and heads that do not divide 32, are stored row by row.
        const bool by_tma = kWarpRows % a.pack == 0 && (a.cu_q == nullptr || it.q0 + (t + 1) * tpt <= it.s.nq);
#pragma unroll 1
        for (int q = 0; q < kCols / 32; ++q) {
          float o[32];
          if (it.n_parts > 1) {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0.f;
#pragma unroll 2
            for (int p = 0; p < it.n_parts; ++p) {
              const float wgt = part_weight(__ldcg(a.part_ml + (slot0 + 2 * p) * kTileM + r).x, m_tot);
              const float4* po = reinterpret_cast<const float4*>(a.part_o + (slot0 + 2 * p) * kTileM * D) + r;
              float4 y[8];
#pragma unroll
              for (int g = 0; g < 8; ++g) y[g] = __ldcg(po + (q * 8 + g) * kTileM);
#pragma unroll
              for (int g = 0; g < 8; ++g) {
                o[4 * g] = fmaf(y[g].x, wgt, o[4 * g]);
                o[4 * g + 1] = fmaf(y[g].y, wgt, o[4 * g + 1]);
                o[4 * g + 2] = fmaf(y[g].z, wgt, o[4 * g + 2]);
                o[4 * g + 3] = fmaf(y[g].w, wgt, o[4 * g + 3]);
              }
            }
          } else {
            uint32_t u[32];
            chunk(q, u);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __uint_as_float(u[i]);
          }
#pragma unroll
          for (int ch = 0; ch < 4; ++ch) {
            const int col = q * 32 + ch * 8;
            const uint32_t addr = stage + (col >> 6) * kBoxBytes + r * 128 + ((((col & 63) >> 3) ^ (r & 7)) << 4);
            const uint32_t w0 = pack2<BF16>(o[ch * 8 + 0] * f, o[ch * 8 + 1] * f);
            const uint32_t w1 = pack2<BF16>(o[ch * 8 + 2] * f, o[ch * 8 + 3] * f);
            const uint32_t w2 = pack2<BF16>(o[ch * 8 + 4] * f, o[ch * 8 + 5] * f);
            const uint32_t w3 = pack2<BF16>(o[ch * 8 + 6] * f, o[ch * 8 + 7] * f);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(w0), "r"(w1), "r"(w2), "r"(w3)
                         : "memory");
          }
          if (by_tma && ((q & 1) || q == kCols / 32 - 1)) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_5d(&tm_o, stage + (q >> 1) * kBoxBytes + (warp & 3) * kWarpRows * 128, (q >> 1) * kBoxCols, 0,
                           static_cast<int>(it.s.row0) + it.q0 + t * tpt + (warp & 3) * div_by(kWarpRows, a.by_pack), it.group,
                           a.cu_q != nullptr ? 0 : it.b);
              tma_store_commit();
            }
          }
        }
        if (by_tma) {
          if (lane == 0) tma_store_wait_read0();  // the staging buffer must outlive the copies' reads
        } else {
          __syncwarp();
          constexpr int kChunks = kCols / 8;  // of 16 bytes in a row
          for (int i = lane; i < kWarpRows * kChunks; i += 32) {
            const int rr = (warp & 3) * kWarpRows + i / kChunks, ch = i % kChunks;
            const int in = div_by(rr, a.by_pack), token = it.q0 + t * tpt + in;
            if (in >= tpt || token >= it.s.nq) continue;
            const uint4 y = *reinterpret_cast<const uint4*>(gbase + L::kOffQ + t * L::kTileBytes + (ch >> 3) * kBoxBytes +
                                                            rr * 128 + (((ch & 7) ^ (rr & 7)) << 4));
            *reinterpret_cast<uint4*>(a.o + it.b * a.os[0] + (it.group * a.pack + (rr - in * a.pack)) * a.os[1] +
                                      (it.s.row0 + token) * a.os[2] + ch * 8) = y;
          }
        }
      }
      tc_fence_before();
    }
  } else {
    reg_dec<kRegOther>();
    if (warp == kWarpMma0 || warp == kWarpMma1) {
      // =========================== MMA issuers =====================================
      // One issuing warp per Q tile, PV_a(j) S_a(j+1) PV_b(j) S_b(j+1); the converged warp walks, an elected thread issues.
      const int t = (warp == kWarpMma0) ? 0 : 1;
      if (n_tiles > 0 && t < nt) {
        const bool issuer = elect_one();
        constexpr uint32_t idesc_s = make_idesc(1, BF16 ? 1 : 0, 0, 0, kTileM, kHalfN);
        constexpr uint32_t idesc_o = make_idesc(1, BF16 ? 1 : 0, 0, 1, kTileM, kCols);
        const uint32_t sQt = sQ + t * L::kTileBytes;
        const uint32_t tO = tmem_base + L::kColO + D * t;
        const uint32_t tSt = tmem_base + L::kColS + 128 * t;
        auto issue_s = [&](int hb, int slot) {  // S(half) = Q_t K[64 * half ..)^T
          if (!issuer) return;
          const uint64_t da = make_smem_desc(sQt, 16, 1024);
          const uint64_t db = make_smem_desc(sRing, 16, 1024) + ((slot * L::kTileBytes + hb * kHalfN * 128) >> 4);
#pragma unroll
          for (int k = 0; k < kCols / 16; ++k) {
            const uint32_t off = ((k / 4) * kBoxBytes + (k % 4) * 32) >> 4;
            mma_f16_ss(tSt + kHalfN * hb, da + off, db + off, idesc_s, k > 0);
          }
        };
        // a slot is free when both Q tiles are done with it; a lone tile's issuer gives both releases
        auto release = [&](int slot) {
          mma_commit(bar(L::kBarKvEmpty + slot));
          if (nt == 1) mma_commit(bar(L::kBarKvEmpty + slot));
        };
        mbar_wait(bar(L::kBarQFull + t), 0, wc, kErrWaitKV);
        mbar_wait(bar(L::kBarKvFull + 0), 0, wc, kErrWaitKV);
        // tile 1 starts when tile 0 has its first row maxima: the two softmax groups then do not want the exp2 unit at the
        // same moments
        if (t == 1) mbar_wait(bar(L::kBarStagger), 0, wc, kErrWaitP);
        tc_fence_after();
        for (int hb = 0; hb < 2; ++hb) {
          issue_s(hb, 0);
          if (issuer) mma_commit(bar(L::kBarSFull + 2 * t + hb));
        }
        if (issuer) release(0);
        __syncwarp();
        int cons = 1;  // ring consumption index: K_0, V_0, K_1, V_1, ...
        for (int j = 0; j < n_tiles; ++j) {
          const int vslot = cons % L::kStages;
          mbar_wait(bar(L::kBarKvFull + vslot), (cons / L::kStages) & 1, wc, kErrWaitKV);
          ++cons;
          const bool has_next = (j + 1 < n_tiles);
          const int kslot = cons % L::kStages;
          const uint32_t kpar = (cons / L::kStages) & 1;
#pragma unroll
          for (int hb = 0; hb < 2; ++hb) {
            mbar_wait(bar(L::kBarPReady + 2 * t + hb), j & 1, wc, kErrWaitP);
            tc_fence_after();
            const uint32_t tP = tSt + kHalfN * hb;
            if (issuer) {
              const uint64_t db = make_smem_desc(sRing, kBoxBytes, 1024) + ((vslot * L::kTileBytes) >> 4);
#pragma unroll
              for (int kk = 0; kk < kHalfN / 16; ++kk) {
                const int k = hb * (kHalfN / 16) + kk;  // 16-key slice of the V tile
                mma_f16_ts(tO, tP + kk * 8, db + k * (2048 >> 4), idesc_o, (j > 0 || k > 0) ? 1u : 0u);
              }
              mma_commit(bar(L::kBarODone + 2 * t + hb));
              if (hb == 1) release(vslot);
            }
            __syncwarp();
            if (has_next) {  // S_h(j+1) after PV_h(j), whose operand P_h(j) lives in the S buffer
              if (hb == 0) {
                mbar_wait(bar(L::kBarKvFull + kslot), kpar, wc, kErrWaitKV);
                tc_fence_after();
              }
              issue_s(hb, kslot);
              if (issuer) {
                mma_commit(bar(L::kBarSFull + 2 * t + hb));
                if (hb == 1) release(kslot);
              }
              __syncwarp();
            }
          }
          if (has_next) ++cons;
        }
      }
      __syncwarp();
    } else if (nt > 0 && n_tiles > 0) {
      // =========================== copies ==========================================
      // Fill i of the ring is K (even) or V (odd) of tile i / 2: warp 9 takes the even ones, warp 11 the odd ones.
      const bool is_v = warp == kWarpV;
      uint32_t raw_phase = 0;
      const int hk = div_by(it.group, a.by_gqa);
      if (is_v) pl.fetch(a, it, it.j0);
      for (int j = is_v ? 0 : 1; j < n_tiles; ++j) {
        const int i = 2 * j + (is_v ? 1 : 0), slot = i % L::kStages, k0 = it.t.at(it.j0 + j) * kTileN;
        pl.settle(a);
        if (j + 1 < n_tiles) pl.fetch(a, it, it.j0 + j + 1);
        if (i >= L::kStages) {
          __nanosleep(200);  // a sleeping warp takes no issue slots from the softmax warps beside it
          mbar_wait(bar(L::kBarKvEmpty + slot), (i / L::kStages - 1) & 1, wc, kErrWaitFree);
        }
        const bool clear = is_v && cache_partly_seen(it.s.lo, it.s.hi, it.s.sink_end, k0, kTileN);
        const uint32_t full = bar(L::kBarKvFull + slot), to = clear ? bar(L::kBarRaw) : full;
        pl.copy(is_v ? &tm_v : &tm_k, sRing + slot * L::kTileBytes, to, hk);
        if (clear) {
          mbar_wait(to, raw_phase, wc, kErrWaitKV);
          raw_phase ^= 1;
          uint8_t* v = gbase + L::kOffRing + slot * L::kTileBytes;
          for (int row = 0; row < kTileN; ++row) {
            if (cache_seen(it.s.lo, it.s.hi, it.s.sink_end, k0 + row, 1)) continue;
            if (lane < 8 * L::kBoxes)
              *reinterpret_cast<uint4*>(v + (lane >> 3) * kBoxBytes + row * 128 + (lane & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(full);
          __syncwarp();
        }
      }
      if (*abort_flag) wait_for_copies();
      __syncwarp();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kWarpMma0) {
    tc_fence_after();
    tmem_dealloc(tmem_base, L::kTmemCols);
  }
}

// ---------------------------------------------------------------------------------
// The rows of a call behind a shared prefix: the pieces that the prefix's launch left and what the launch over the rest of
// each sequence left, added up and stored.  A warp takes 32 rows of a Q tile and 4 columns of them, a lane a row.  Bound: the
// loads that wait for one another, so a running maximum instead of a pass over the pieces for it, and kAhead pieces together.
template <int D, bool BF16>
__global__ void __launch_bounds__(128)
cache_merge_kernel(const CacheArgs a, int n_parts) {
  grid_dep_launch();
  grid_dep_wait();
  const int r = threadIdx.x, t = blockIdx.x & 1, col = blockIdx.y * 4;
  const int item = blockIdx.x >> 1, idx = div_by(item, a.by_groups), group = item - idx * a.groups;
  const int in_tile = div_by(r, a.by_pack), tok = (2 * (a.pairs - 1 - idx) + t) * a.tpt + in_tile;
  const int head = group * a.pack + (r - in_tile * a.pack);
  const int rows = a.cu_q != nullptr ? a.total_q : a.B * a.Nq;
  if (in_tile >= a.tpt || tok >= rows) return;
  if (a.cu_q != nullptr && (tok < a.cu_q[0] || tok >= a.cu_q[a.B])) return;  // no sequence's
  const long long rest = static_cast<long long>(tok) * a.Hq + head;
  const float2 ml_rest = a.rest_ml[rest];
  const float4 y_rest = *reinterpret_cast<const float4*>(a.rest_o + rest * D + col);
  float m = ml_rest.x, l = ml_rest.y, o[4] = {y_rest.x, y_rest.y, y_rest.z, y_rest.w};
  // A row without keys in the rest: its sum is 0.  A row maximum of -inf does not say so: that of the launch over the rest
  // passes over NaN, and a row all of whose keys score one has it beside a sum that is NaN.
  if (l == 0.f) o[0] = o[1] = o[2] = o[3] = 0.f;
  constexpr int kAhead = 16;  // pieces whose loads are in flight together
  for (int p0 = 0; p0 < n_parts; p0 += kAhead) {
    float4 y[kAhead];
    float2 ml[kAhead];
    float top = m;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (p0 + u >= n_parts) break;
      const long long at = ((static_cast<long long>(item) * n_parts + p0 + u) * 2 + t) * kTileM + r;
      ml[u] = a.part_ml[at];
      y[u] = *(reinterpret_cast<const float4*>(a.part_o + (at - r) * D) + (col / 4) * kTileM + r);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (p0 + u < n_parts) top = fmaxf(top, ml[u].x);
    const float keep = part_weight(m, top);
    m = top;
    l *= keep;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] *= keep;
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      // A piece of which the row sees no key is left out, not weighted with 0: its O is 0 times the values that other sequences
      // see, which an infinity or a NaN among them makes a NaN.
      if (p0 + u < n_parts && ml[u].y != 0.f) {
        const float w = part_weight(ml[u].x, m);
        l = fmaf(ml[u].y, w, l);
        o[0] = fmaf(y[u].x, w, o[0]);
        o[1] = fmaf(y[u].y, w, o[1]);
        o[2] = fmaf(y[u].z, w, o[2]);
        o[3] = fmaf(y[u].w, w, o[3]);
      }
  }
  const float f = l > 0.f ? 1.f / l : l;  // a NaN stays one
  long long seq = 0, at = tok;
  if (a.cu_q == nullptr) {
    seq = div_by(tok, a.by_nq);
    at = tok - seq * a.Nq;
  }
  *reinterpret_cast<uint2*>(a.o + seq * a.os[0] + head * a.os[1] + at * a.os[2] + col) =
      make_uint2(pack2<BF16>(o[0] * f, o[1] * f), pack2<BF16>(o[2] * f, o[3] * f));
  if (col == 0 && a.lse != nullptr) a.lse[seq * a.ls[0] + head * a.ls[1] + at] = row_lse(m, l);
}

template <int D, bool BF16, bool PREFIX, bool NARROW = false>
static cudaError_t launch_t(const CUtensorMap* tm, const CacheArgs& a, int ctas, int parts, cudaStream_t st) {
  auto kern = fwd_cache_ws_kernel<D, BF16, PREFIX, NARROW>;
  static std::atomic<unsigned long long> smem_set{0};
  cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void*>(kern), Layout<D>::kDynSmem, &smem_set);
  if (e != cudaSuccess) return e;
  return launch_overlapped(kern, dim3(ctas, parts), kThreads, Layout<D>::kDynSmem, st, tm[0], tm[1], tm[2], tm[3], a);
}

template <int D, bool BF16>
static cudaError_t launch_d(bool prefix, const CUtensorMap* tm, const CacheArgs& a, int items, int parts, cudaStream_t st) {
  if constexpr (D == 128) {
    if (a.D == 96) {
      if (prefix) return launch_t<D, BF16, true, true>(tm, a, items, parts, st);
      return launch_t<D, BF16, false, true>(tm, a, items, parts, st);
    }
  }
  return prefix ? launch_t<D, BF16, true>(tm, a, items, parts, st) : launch_t<D, BF16, false>(tm, a, items, parts, st);
}

// tm: Q (5-D, boxes of tpt tokens x pack heads), K, V (boxes of 64 columns x min(128, page size) keys), O (5-D, boxes of a
// warp's 32 rows).  a.pair_items pairs of Q tiles x groups of heads, the rest of the `ctas` a Q tile each, all cut into at most
// `parts` pieces; ragged: as many CTAs as there may be pieces.
cudaError_t launch_fwd_cache_ws(int D, bool bf16, bool prefix, const CUtensorMap* tm, const CacheArgs& a, int items, int parts,
                                cudaStream_t st) {
  if (D == 128)
    return bf16 ? launch_d<128, true>(prefix, tm, a, items, parts, st) : launch_d<128, false>(prefix, tm, a, items, parts, st);
  if (D == 64)
    return bf16 ? launch_d<64, true>(prefix, tm, a, items, parts, st) : launch_d<64, false>(prefix, tm, a, items, parts, st);
  return cudaErrorInvalidValue;
}

// After launch_fwd_cache_ws over the prefix (`items` x `parts` pieces) and launch_fwd_cache over the rest.
cudaError_t launch_cache_merge(int D, bool bf16, const CacheArgs& a, int items, int parts, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(items) * 2, a.D / 4);
  if (D == 128)
    return bf16 ? launch_overlapped(cache_merge_kernel<128, true>, grid, 128, 0, st, a, parts)
                : launch_overlapped(cache_merge_kernel<128, false>, grid, 128, 0, st, a, parts);
  if (D == 64)
    return bf16 ? launch_overlapped(cache_merge_kernel<64, true>, grid, 128, 0, st, a, parts)
                : launch_overlapped(cache_merge_kernel<64, false>, grid, 128, 0, st, a, parts);
  return cudaErrorInvalidValue;
}

}  // namespace ma
