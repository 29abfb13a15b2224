// Attention over a cache for few query rows per KV head (decode, drafts), and for any others.
//
// o_i = sum_j p_ij v_j / sum_j p_ij with p_ij = exp(s_ij - m_i) over the keys j that query token i sees: those up to its
// own position, at most the last `window` of them and the first `sinks` ones.  K and V come through a block table (pages
// of 16 to 1024 tokens in any order) or lie one after the other.  One pass over the keys with a running maximum and sum.
//
//   item      = (sequence, KV head, block of 16 * RG rows); a row is (token, query head of the KV head's G), so that K and V
//               cross an SM once for all the heads that share them
//   CTA       = a contiguous range of the 64-key tiles of all items, the same length for each (an item counts kItemCost tiles
//               more: dealt out by tiles alone, 512 items of 1 to 16 tiles took 26.5 instead of 21.3 us, cold); lengths are
//               known on the GPU alone, so every CTA adds up the tiles of all sequences and finds its own
//   warp 4    TMA producer: a copy per page (at most 64 keys) and 64 columns of K and of V, each issued by a lane of its own
//   warps 0-3 16 rows x (16 * RG keys of the tile) each, running (m, l, O) in registers
//
// A CTA whose range cuts an item leaves its piece (un-normalised O, m, l) in scratch and counts itself in; the one that
// counts in last folds the pieces.  Behind a shared prefix the rows are left un-normalised for the launch that adds its pieces.
//
// Bound: HBM where the contexts are long: 16 requests of 1001 to 16001 keys, 32/8 heads of 128, pages of 16 tokens 67.5 us = 5.6
// TB/s, 0.85 of the measured copy rate; 32 with a window of 4096 90 us = 5.8 TB/s, 0.89.  The registers of two CTAs an SM: 32
// bytes spill at D = 128 with one row group.  Short calls are bound by their chain of
// loads: lengths (0.7 us), the walk to the CTA's range (0.8), block table and first tile (1.2), half a microsecond a tile, 0.5
// to leave a piece and 3 to fold: 4 requests of 100 to 1000 keys, 12 heads of 64 9 us (pieces of 4 tiles; of 6, 8 and 12: 9.5,
// 10.1, 11.9, with an earlier fold).
//
// Keys that no row sees are never read: their pages may be gone or hold anything.  Where a tile holds some, their scores
// are replaced and their rows of V cleared, so that what lies there does not reach a result.
#include <atomic>
#include <type_traits>

#include "cache.cuh"
#include "launch.cuh"
#include "mma_sync.cuh"
#include "ptx.cuh"

namespace ma {

namespace {

constexpr int kThreads = 160;
constexpr int kKeys = 64;            // keys per tile
constexpr int kBox = kKeys * 128;    // one [64 keys x 128 B] box
constexpr float kLazy = 8.0f;        // log2 units a row's maximum may move before O is rescaled
constexpr int kMergePitch = 36;      // floats per row of the merge buffer (32 + padding)
constexpr int kPiece = 4;            // tiles of a piece where every CTA works on one
constexpr int kItemCost = 3;         // what an item takes beside its tiles, in tiles

template <int D>
struct Layout {
  static constexpr int kBoxes = D / 64;
  static constexpr int kStageBytes = 2 * kBoxes * kBox;  // K then V
  static constexpr int kStages = D == 64 ? 4 : 3;
  static constexpr int kOffMerge = kStages * kStageBytes;              // float[4 warps][16][kMergePitch]
  static constexpr int kOffMl = kOffMerge + 4 * 16 * kMergePitch * 4;  // float2[4 warps][16]
  static constexpr int kOffBar = kOffMl + 4 * 16 * 8;                  // full[kStages], empty[kStages]
  static constexpr int kOffScan = kOffBar + 2 * kStages * 8;           // long long[2][4 warps], tiles before the first sequence
  static constexpr int kOffWalk = kOffScan + 10 * 8;                   // Walk of the first sequence
  static constexpr int kOffMisc = kOffWalk + 80;                       // abort flag, arrival order, first sequence
  static constexpr int kBytes = kOffMisc + 16;
  static constexpr int kDynSmem = kBytes + 1024;
};

__device__ __forceinline__ void workers_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// weight of a partial with maximum m under the total maximum mt (0 for a partial without keys)
__device__ __forceinline__ float part_weight(float m, float mt) { return m == -INFINITY ? 0.f : ex2(m - mt); }
// natural logarithm of a row's sum; -inf where it saw no key, NaN where a score was one
__device__ __forceinline__ float row_lse(float m, float l) {
  return l == 0.f ? -INFINITY : m * 0.6931471805599453f + __logf(l);
}

// Sequence b of the call, and how its items are counted: n_rb row blocks per KV head, `slots` places on the launch's line for
// each: its t.n tiles and kItemCost more for its start and end, or, where a launch is so short that every CTA works on one
// piece, what fills the last piece up.
struct Walk {
  CacheSeq s;
  CacheTiles t;
  int n_rb, slots;
  __device__ __forceinline__ long long total(const CacheArgs& a) const {
    return static_cast<long long>(a.Hkv) * n_rb * slots;
  }
};
static_assert(sizeof(Walk) <= 80, "Walk");
template <int kRows>
__device__ __forceinline__ Walk walk_to(const CacheArgs& a, int b, bool pieces) {
  Walk w;
  int r0 = 0, r1 = 0;
  if (a.cu_q != nullptr) {
    r0 = a.cu_q[b];
    r1 = a.cu_q[b + 1];
  }
  w.s = cache_seq(a, r0, r1, a.seq_lens != nullptr ? a.seq_lens[b] : 0);
  w.t = cache_tiles<kKeys>(w.s.lo, w.s.hi, w.s.sink_end);
  w.n_rb = static_cast<int>((static_cast<long long>(w.s.nq) * a.G + kRows - 1) / kRows);
  w.slots = pieces ? (w.t.n + (kPiece - 1)) / kPiece * kPiece : w.t.n + kItemCost;
  return w;
}

}  // namespace

template <int D, bool BF16, int RG>
__global__ void __launch_bounds__(kThreads, 2)
fwd_cache_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const CacheArgs a) {
  using L = Layout<D>;
  constexpr int KG = 4 / RG;      // key groups: warps that share a row group
  constexpr int kRows = 16 * RG;  // rows of an item
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t sbase = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (sbase - raw);
  const uint32_t bars = sbase + L::kOffBar;
  auto full = [&](int s) -> uint32_t { return bars + 8u * s; };
  auto empty = [&](int s) -> uint32_t { return bars + 8u * (L::kStages + s); };
  long long* scan = reinterpret_cast<long long*>(gbase + L::kOffScan);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gbase + L::kOffMisc);
  volatile int* order = abort_flag + 1;
  int* first_seq = reinterpret_cast<int*>(gbase + L::kOffMisc) + 2;

  grid_dep_launch();
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const WaitCtx wc{abort_flag, a.status, MINIATTN_WAIT_LIMIT_NS};
  if (tid == 128) {
    for (int s = 0; s < L::kStages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 4);
    }
    *abort_flag = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
  }
  grid_dep_wait();

  // ---- this CTA's tiles [lo, hi) of the launch's total: each of 128 threads adds up a run of sequences.  Where pieces of
  // kPiece tiles, none with tiles of two items, are no more than the CTAs, each CTA takes one; otherwise all tiles are cut
  // alike. ----
  const int run = (a.B + 127) / 128;
  const int b0 = min(a.B, tid * run), b1 = tid < 128 ? min(a.B, b0 + run) : b0;
  long long mine = 0, mine_pieces = 0;
  bool bad = false;
  Walk own{};
  for (int b = b0; b < b1; ++b) {
    const Walk w = walk_to<kRows>(a, b, true);
    const long long items = static_cast<long long>(a.Hkv) * w.n_rb;
    mine += items * (w.t.n + kItemCost);
    mine_pieces += items * w.slots;
    bad |= w.s.bad;
    if (run == 1) own = w;
  }
  if (bad && a.status != nullptr) atomicOr(a.status, kErrCache);
  long long before = mine, before_pieces = mine_pieces;  // inclusive over the warp, then exclusive over the CTA
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, before, d), op = __shfl_up_sync(0xffffffffu, before_pieces, d);
    if (lane >= d) {
      before += o;
      before_pieces += op;
    }
  }
  if (lane == 31 && warp < 4) {
    scan[warp] = before;
    scan[4 + warp] = before_pieces;
  }
  __syncthreads();
  long long total = 0, total_pieces = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < warp) {
      before += scan[w];
      before_pieces += scan[4 + w];
    }
    total += scan[w];
    total_pieces += scan[4 + w];
  }
  const long long n_ctas = gridDim.x;
  const bool pieces = total_pieces <= n_ctas * kPiece;
  const long long share = pieces ? kPiece : cache_div(total + n_ctas - 1, n_ctas);
  if (pieces) {
    total = total_pieces;
    before = before_pieces;
    mine = mine_pieces;
  }
  before -= mine;
  const long long lo = blockIdx.x * share, hi = min(total, lo + share);
  if (lo >= hi) return;
  if (tid < 128 && lo >= before && lo < before + mine) {
    int b = b0;
    if (run == 1) {
      if (!pieces) own.slots = own.t.n + kItemCost;
    } else {
      for (;; ++b) {
        own = walk_to<kRows>(a, b, pieces);
        const long long n = own.total(a);
        if (lo < before + n || b + 1 >= b1) break;
        before += n;
      }
    }
    *first_seq = b;
    scan[8] = before;
    *reinterpret_cast<Walk*>(gbase + L::kOffWalk) = own;
  }
  __syncthreads();
  int b = *first_seq;
  long long base = scan[8];  // places before sequence b
  Walk w = *reinterpret_cast<const Walk*>(gbase + L::kOffWalk);
  auto next_seq = [&]() {  // the next sequence that has rows; only while places are left
    do {
      base += w.total(a);
      b = min(b + 1, a.B - 1);
      w = walk_to<kRows>(a, b, pieces);
    } while (w.n_rb == 0 && b + 1 < a.B);
  };

  if (warp == 4) {
    // =========================== TMA producer ====================================
    // Lane l copies one box of a tile: page l / (2 * kBoxes) of it, K or V, 64 columns.  The page numbers of the next tile
    // are fetched before the wait for its slot.
    const int keys_shift = a.table != nullptr ? min(6, a.page_shift) : 6;  // keys of a box
    const int n_lanes = (kKeys >> keys_shift) * 2 * L::kBoxes;
    const int sub = lane / (2 * L::kBoxes), bx = lane % L::kBoxes;
    const bool is_v = (lane / L::kBoxes) & 1;
    const uint32_t dst = (is_v ? L::kBoxes * kBox : 0) + bx * kBox + ((sub << keys_shift) << 7);
    const CUtensorMap* tm = is_v ? &tm_v : &tm_k;
    const uint32_t box_bytes = 128u << keys_shift;
    const long long it0 = cache_div(lo - base, w.slots);
    int j = static_cast<int>(lo - base - it0 * w.slots);
    int hk = static_cast<int>(cache_div(it0, w.n_rb)), rb = static_cast<int>(it0 - static_cast<long long>(hk) * w.n_rb);
    int key = 0, page = 0;
    bool wanted = false;
    auto look_up = [&]() {  // the page of this lane's keys of tile j
      key = w.t.at(j) * kKeys + (sub << keys_shift);
      wanted = lane < n_lanes && cache_seen(w.s.lo, w.s.hi, w.s.sink_end, key, 1 << keys_shift);
      page = b;
      if (a.table != nullptr) {
        if (wanted) page = a.table[b * a.table_stride + (key >> a.page_shift)];
        key &= (1 << a.page_shift) - 1;
        if (wanted && static_cast<unsigned>(page) >= static_cast<unsigned>(a.n_pages)) {
          wanted = false;
          if (a.status != nullptr) atomicOr(a.status, kErrCache);
        }
      }
    };
    long long x = lo;
    auto to_a_tile = [&]() {  // past the places of items that hold no tile
      while (x < hi && j >= w.t.n) {
        x += w.slots - j;
        j = 0;
        if (x < hi && ++rb == w.n_rb) {
          rb = 0;
          if (++hk == a.Hkv) {
            hk = 0;
            next_seq();
          }
        }
      }
    };
    to_a_tile();
    if (x < hi) look_up();
    int slot = 0, par = 1;
    for (int i = 0; x < hi; ++i) {
      if (i >= L::kStages) mbar_wait(empty(slot), par, wc, kErrWaitFree);
      const uint32_t n_copies = __popc(__ballot_sync(0xffffffffu, wanted));
      if (lane == 0) mbar_expect_tx(full(slot), n_copies * box_bytes);
      __syncwarp();
      if (wanted) tma_load_4d(sbase + slot * L::kStageBytes + dst, tm, full(slot), bx * 64, key, hk, page);
      __syncwarp();
      if (++slot == L::kStages) {
        slot = 0;
        par ^= 1;
      }
      ++x;
      ++j;
      to_a_tile();
      if (x < hi) look_up();
    }
    // give-up path: let the copies in flight land (bounded) before the shared memory is released
    if (*abort_flag) {
      const uint64_t t0 = global_timer_ns();
      while (global_timer_ns() - t0 < 2000000ull) {
      }
    }
    __syncwarp();
    return;
  }

  // ---------------------------------------------------------------- workers
  const int rg = warp % RG, kg = warp / RG;
  const int g = lane >> 2, tig = lane & 3;
  float* merge = reinterpret_cast<float*>(gbase + L::kOffMerge);
  float2* ml_s = reinterpret_cast<float2*>(gbase + L::kOffMl);
  const float c = a.scale_log2;
  // ldmatrix row addresses: lanes 0-7 / 8-15 / 16-23 / 24-31 address the four 8x8 matrices
  const int k_row = (lane & 7) + ((lane >> 4) << 3), k_chunk = (lane >> 3) & 1;  // K: keys x dims
  const int v_row = (lane & 7) + (((lane >> 3) & 1) << 3), v_chunk = lane >> 4;  // V: trans
  int slot = 0, par = 0;

  for (long long x = lo; x < hi;) {
    while (x >= base + w.total(a) && b + 1 < a.B) next_seq();
    const long long it = cache_div(x - base, w.slots);
    const long long item0 = base + it * w.slots;
    const int t0 = static_cast<int>(x - item0);
    const int t1 = static_cast<int>(min(static_cast<long long>(w.t.n), hi - item0));
    if (t0 >= w.t.n) {  // places that hold no tile
      x = item0 + w.slots;
      continue;
    }
    const int hk = static_cast<int>(cache_div(it, w.n_rb)), rb = static_cast<int>(it - static_cast<long long>(hk) * w.n_rb);
    if (hk >= a.Hkv) break;  // only if the lengths changed under the launch
    const int rows = w.s.nq * a.G, row0 = rb * kRows;

    // Q fragments of this warp's 16 rows, and which keys its two rows of this lane see
    uint32_t qf[D / 16][4];
    int first[2], end[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = row0 + rg * 16 + g + 8 * e;
      const int tok = div_by(r, a.by_g);
      const bool ok = r < rows;
      cache_row(a, w.s, tok, &first[e], &end[e]);
      if (!ok) end[e] = 0;
      const uint16_t* qp = a.q + b * a.qs[0] + (hk * a.G + (r - tok * a.G)) * a.qs[1] + (w.s.row0 + tok) * a.qs[2];
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const int col = ks * 16 + tig * 2;  // D = 96 runs on the D = 128 kernel: columns past it are 0
        qf[ks][e] = (ok && col < a.D) ? *reinterpret_cast<const uint32_t*>(qp + col) : 0u;
        qf[ks][2 + e] = (ok && col + 8 < a.D) ? *reinterpret_cast<const uint32_t*>(qp + col + 8) : 0u;
      }
    }
    const int all_from = __reduce_max_sync(0xffffffffu, max(first[0], first[1]));
    const int all_to = __reduce_min_sync(0xffffffffu, min(end[0], end[1]));

    float acc[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};

    for (int t = t0; t < t1; ++t) {
      mbar_wait(full(slot), par, wc, kErrWaitKV);
      const uint32_t sK = sbase + slot * L::kStageBytes;
      const uint32_t sV = sK + L::kBoxes * kBox;
      const int key0 = kg * kRows;  // this warp's keys of the tile: [key0, key0 + 16 * RG)
      const int kbase = w.t.at(t) * kKeys + key0;
      const bool some_hidden = kbase < all_from || kbase + kRows > all_to;
      if (kbase + kRows > w.s.hi || kbase < w.s.lo) {
        // Keys that no row sees: whatever lies in their rows of V (another sequence's, nothing yet, an infinity) must not
        // meet their weight of 0.  Warps that share the keys write the same zeros.
        uint8_t* rows_v = gbase + slot * L::kStageBytes + L::kBoxes * kBox;
        for (int i = lane; i < kRows * 8 * L::kBoxes; i += 32) {
          const int r = (i >> 3) % kRows, box = (i >> 3) / kRows;
          if (!cache_seen(w.s.lo, w.s.hi, w.s.sink_end, kbase + r, 1))
            *reinterpret_cast<uint4*>(rows_v + box * kBox + (key0 + r) * 128 + (i & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();  // the slot's next copy comes after these writes
        __syncwarp();
      }
      // All RG * 2 accumulator chains advance together, and with one row group each is cut in two: an mma.sync waits for
      // the one before it on its chain.
      constexpr int kSplit = RG == 1 ? 2 : 1;
      float sp[kSplit][RG][2][4];
#pragma unroll
      for (int u = 0; u < kSplit; ++u)
#pragma unroll
        for (int kc = 0; kc < RG; ++kc)
#pragma unroll
          for (int e = 0; e < 4; ++e) sp[u][kc][0][e] = sp[u][kc][1][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
#pragma unroll
        for (int kc = 0; kc < RG; ++kc) {
          const int r = key0 + kc * 16 + k_row;
          uint32_t kb[4];
          ldsm4(sK + r * 128 + (ks >> 2) * kBox + ((((ks & 3) * 2 + k_chunk) ^ (r & 7)) << 4), kb);
          mma16816<BF16>(sp[ks % kSplit][kc][0], qf[ks], kb[0], kb[1]);
          mma16816<BF16>(sp[ks % kSplit][kc][1], qf[ks], kb[2], kb[3]);
        }
      }
      auto& s = sp[0];
      if constexpr (kSplit == 2) {
#pragma unroll
        for (int kc = 0; kc < RG; ++kc)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[kc][0][e] += sp[kSplit - 1][kc][0][e];
            s[kc][1][e] += sp[kSplit - 1][kc][1][e];
          }
      }
      if (some_hidden) {  // by selection: what a hidden key's score holds does not matter
#pragma unroll
        for (int kc = 0; kc < RG; ++kc)
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = kbase + kc * 16 + n * 8 + tig * 2 + (e & 1);
              if (key >= end[e >> 1] || (key < first[e >> 1] && key >= a.sinks)) s[kc][n][e] = -INFINITY;
            }
      }
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int kc = 0; kc < RG; ++kc)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          mx[0] = fmax3(mx[0], s[kc][n][0], s[kc][n][1]);
          mx[1] = fmax3(mx[1], s[kc][n][2], s[kc][n][3]);
        }
      bool moved = false;
      float alpha[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2)) * c;
        const float m_new = fmaxf(m_run[e], mx[e]);
        alpha[e] = 1.f;
        if (m_new - m_run[e] > kLazy) {  // also taken when the running maximum is -inf
          alpha[e] = ex2(m_run[e] - m_new);
          m_run[e] = m_new;
          moved = true;
        }
      }
      if (__any_sync(0xffffffffu, moved)) {
        l_run[0] *= alpha[0];
        l_run[1] *= alpha[1];
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          acc[n][0] *= alpha[0];
          acc[n][1] *= alpha[0];
          acc[n][2] *= alpha[1];
          acc[n][3] *= alpha[1];
        }
      }
      const float mc0 = m_run[0] == -INFINITY ? 0.f : m_run[0];
      const float mc1 = m_run[1] == -INFINITY ? 0.f : m_run[1];
#pragma unroll
      for (int kc = 0; kc < RG; ++kc) {
        uint32_t pf[4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float p0 = ex2(fmaf(s[kc][n][0], c, -mc0)), p1 = ex2(fmaf(s[kc][n][1], c, -mc0));
          const float p2 = ex2(fmaf(s[kc][n][2], c, -mc1)), p3 = ex2(fmaf(s[kc][n][3], c, -mc1));
          l_run[0] += p0 + p1;
          l_run[1] += p2 + p3;
          // P in 16 bits for the second product: off by half a step of the type for each weight
          pf[2 * n] = pack2<BF16>(p0, p1);
          pf[2 * n + 1] = pack2<BF16>(p2, p3);
        }
        const int r = key0 + kc * 16 + v_row;
        const uint32_t rowa = sV + r * 128;
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
          uint32_t vb[4];
          ldsm4_t(rowa + (n >> 2) * kBox + ((((n & 3) * 2 + v_chunk) ^ (r & 7)) << 4), vb);
          mma16816<BF16>(acc[2 * n], pf, vb[0], vb[1]);
          mma16816<BF16>(acc[2 * n + 1], pf, vb[2], vb[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty(slot));
      if (++slot == L::kStages) {
        slot = 0;
        par ^= 1;
      }
    }

    // ---- end of a piece: fold the key groups, then write the rows or publish the partial ----
    const bool whole = t0 == 0 && t1 == w.t.n;
    const bool rest = a.rest_o != nullptr;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 1);
      l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 2);
      if (tig == 0) ml_s[warp * 16 + g + 8 * e] = make_float2(m_run[e], l_run[e]);
    }
    workers_sync();
    float f[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float mt = -INFINITY, lt = 0.f;
#pragma unroll
      for (int k = 0; k < KG; ++k) mt = fmaxf(mt, ml_s[(k * RG + rg) * 16 + g + 8 * e].x);
#pragma unroll
      for (int k = 0; k < KG; ++k) {
        const float2 ml = ml_s[(k * RG + rg) * 16 + g + 8 * e];
        lt += ml.y * part_weight(ml.x, mt);
      }
      f[e] = part_weight(m_run[e], mt);
      if (whole && !rest) f[e] *= lt > 0.f ? 1.f / lt : lt;  // a NaN stays one
    }
    const long long c_first = cache_div(item0, share);  // CTA that holds the item's first tile
    const long long my_slot = 2ll * blockIdx.x + (t0 == 0 ? 1 : 0);
    auto lse_at = [&](int r) -> float* {
      const int tok = div_by(r, a.by_g), h = hk * a.G + (r - tok * a.G);
      return a.lse + b * a.ls[0] + h * a.ls[1] + w.s.row0 + tok;
    };
    auto rest_row = [&](int r) -> long long {
      const int tok = div_by(r, a.by_g), h = hk * a.G + (r - tok * a.G);
      return ((a.cu_q != nullptr ? w.s.row0 : static_cast<long long>(b) * a.Nq) + tok) * a.Hq + h;
    };
    if (tid < kRows && row0 + tid < rows) {
      const int rgi = tid >> 4, rr = tid & 15;
      float mt = -INFINITY, lt = 0.f;
      for (int k = 0; k < KG; ++k) mt = fmaxf(mt, ml_s[(k * RG + rgi) * 16 + rr].x);
      for (int k = 0; k < KG; ++k) {
        const float2 ml = ml_s[(k * RG + rgi) * 16 + rr];
        lt += ml.y * part_weight(ml.x, mt);
      }
      if (!whole) a.part_ml[my_slot * kRows + tid] = make_float2(mt, lt);
      else if (rest) a.rest_ml[rest_row(row0 + tid)] = make_float2(mt, lt);
      else if (a.lse != nullptr) *lse_at(row0 + tid) = row_lse(mt, lt);
    }
    auto store_row = [&](int r_in, int col, const float4& o) {  // four columns of a finished row
      if (rest) {
        *reinterpret_cast<float4*>(a.rest_o + rest_row(row0 + r_in) * D + col) = o;
        return;
      }
      if (col >= a.D) return;
      const int r = row0 + r_in, tok = div_by(r, a.by_g), h = hk * a.G + (r - tok * a.G);
      uint2 y;
      y.x = pack2<BF16>(o.x, o.y);
      y.y = pack2<BF16>(o.z, o.w);
      *reinterpret_cast<uint2*>(a.o + b * a.os[0] + h * a.os[1] + (w.s.row0 + tok) * a.os[2] + col) = y;
    };
    if (RG == 1 && rows - row0 <= 4) {
      // the four key groups of at most four rows fit the buffer at once: [warp][4 rows][D]
      if (g < 4) {
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
          *reinterpret_cast<float2*>(merge + (warp * 4 + g) * (D + 4) + n * 8 + tig * 2) =
              make_float2(acc[n][0] * f[0], acc[n][1] * f[0]);
      }
      workers_sync();
      const int r_in = tid / (D / 4), col = (tid % (D / 4)) * 4;
      for (int rr = r_in; rr < rows - row0; rr += 512 / D) {
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < KG; ++k) {
          const float4 y = *reinterpret_cast<const float4*>(merge + (k * 4 + rr) * (D + 4) + col);
          o.x += y.x;
          o.y += y.y;
          o.z += y.z;
          o.w += y.w;
        }
        if (!whole) *reinterpret_cast<float4*>(a.part_o + (my_slot * kRows + rr) * D + col) = o;
        else store_row(rr, col, o);
      }
      workers_sync();
    } else {
#pragma unroll
      for (int p = 0; p < D / 32; ++p) {  // 32 columns at a time through 9 KB
        float* mine_s = merge + warp * 16 * kMergePitch;
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
          const int n = p * 4 + jj;
          *reinterpret_cast<float2*>(mine_s + g * kMergePitch + jj * 8 + tig * 2) =
              make_float2(acc[n][0] * f[0], acc[n][1] * f[0]);
          *reinterpret_cast<float2*>(mine_s + (g + 8) * kMergePitch + jj * 8 + tig * 2) =
              make_float2(acc[n][2] * f[1], acc[n][3] * f[1]);
        }
        workers_sync();
        const int rr = tid >> 3, c4 = (tid & 7) * 4;
#pragma unroll
        for (int rgi = 0; rgi < RG; ++rgi) {
          const int r_in = rgi * 16 + rr;
          if (row0 + r_in >= rows) continue;
          float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int k = 0; k < KG; ++k) {
            const float4 y = *reinterpret_cast<const float4*>(merge + ((k * RG + rgi) * 16 + rr) * kMergePitch + c4);
            o.x += y.x;
            o.y += y.y;
            o.z += y.z;
            o.w += y.w;
          }
          const int col = p * 32 + c4;
          if (!whole) *reinterpret_cast<float4*>(a.part_o + (my_slot * kRows + r_in) * D + col) = o;
          else store_row(r_in, col, o);
        }
        workers_sync();
      }
    }
    if (!whole) {
      __threadfence();  // release: the piece before the count
      workers_sync();
      const int n_parts = static_cast<int>(cache_div(item0 + w.t.n - 1, share) - c_first + 1);
      if (tid == 0) {
        __threadfence();
        *order = atomicAdd(a.counters + c_first, 1);
      }
      workers_sync();
      if (*order == n_parts - 1) {
        __threadfence();  // acquire: every other piece was published before it was counted
        if (tid == 0) a.counters[c_first] = 0;
        const int n_rows = min(kRows, rows - row0);
        // where the pieces of a row lie: the first, the others two slots apart
        auto piece = [&](int p, int r_in) { return (2 * (c_first + p) + (p == 0 ? 1 : 0)) * kRows + r_in; };
        // Four columns of a row per thread, the loads of several pieces in flight together (eight at D = 128 spill: 67.6 -> 69.6 us
        // for 16 long contexts).
        constexpr int kAhead = RG == 1 && D == 64 ? 8 : 4;
        const int n_el = n_rows * (D / 4);
        for (int e = tid; e < n_el; e += 128) {
          const int r_in = e / (D / 4), col = (e % (D / 4)) * 4;
          float mt = -INFINITY, lt = 0.f;
          float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int p0 = 0; p0 < n_parts; p0 += kAhead) {
            float2 ml[kAhead];
            float4 y[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
              if (p0 + u >= n_parts) break;
              const long long i = piece(p0 + u, r_in);
              ml[u] = __ldcg(a.part_ml + i);
              y[u] = __ldcg(reinterpret_cast<const float4*>(a.part_o + i * D + col));
            }
            float top = mt;
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
              if (p0 + u < n_parts) top = fmaxf(top, ml[u].x);
            const float kept = part_weight(mt, top);
            lt *= kept;
            o.x *= kept;
            o.y *= kept;
            o.z *= kept;
            o.w *= kept;
            mt = top;
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
              if (p0 + u >= n_parts) break;
              const float wgt = part_weight(ml[u].x, mt);
              lt = fmaf(ml[u].y, wgt, lt);
              o.x = fmaf(y[u].x, wgt, o.x);
              o.y = fmaf(y[u].y, wgt, o.y);
              o.z = fmaf(y[u].z, wgt, o.z);
              o.w = fmaf(y[u].w, wgt, o.w);
            }
          }
          const float inv = rest ? 1.f : lt > 0.f ? 1.f / lt : lt;
          o.x *= inv;
          o.y *= inv;
          o.z *= inv;
          o.w *= inv;
          store_row(r_in, col, o);
          if (col == 0) {
            if (rest) a.rest_ml[rest_row(row0 + r_in)] = make_float2(mt, lt);
            else if (a.lse != nullptr) *lse_at(row0 + r_in) = row_lse(mt, lt);
          }
        }
      }
      workers_sync();  // `order` may be written again only when everyone has read it
    }
    x = item0 + (t1 == w.t.n ? w.slots : t1);
  }
}

// ---------------------------------------------------------------------------------
template <int D, bool BF16, int RG>
static cudaError_t launch_t(const CUtensorMap* tm, const CacheArgs& a, int n_ctas, cudaStream_t st) {
  auto kern = fwd_cache_kernel<D, BF16, RG>;
  static std::atomic<unsigned long long> smem_set{0};
  cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void*>(kern), Layout<D>::kDynSmem, &smem_set);
  if (e != cudaSuccess) return e;
  return launch_overlapped(kern, n_ctas, kThreads, Layout<D>::kDynSmem, st, tm[0], tm[1], a);
}

template <int D, bool BF16>
static cudaError_t launch_d(const CUtensorMap* tm, const CacheArgs& a, int rg, int n_ctas, cudaStream_t st) {
  if (rg == 1) return launch_t<D, BF16, 1>(tm, a, n_ctas, st);
  return launch_t<D, BF16, 2>(tm, a, n_ctas, st);
}

// tm[0], tm[1]: K and V maps with boxes of 64 columns x min(64, page size) keys.
cudaError_t launch_fwd_cache(int D, bool bf16, const CUtensorMap* tm, const CacheArgs& a, int rg, int n_ctas,
                             cudaStream_t st) {
  if (D == 128) return bf16 ? launch_d<128, true>(tm, a, rg, n_ctas, st) : launch_d<128, false>(tm, a, rg, n_ctas, st);
  if (D == 64) return bf16 ? launch_d<64, true>(tm, a, rg, n_ctas, st) : launch_d<64, false>(tm, a, rg, n_ctas, st);
  return cudaErrorInvalidValue;
}

}  // namespace ma
