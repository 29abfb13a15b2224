// New tokens into a paged cache, rotated by their positions on the way.
//
// With the angle t_i = pos * theta^(-2i / rot) of pair i, (x, y) becomes (x cos t_i - y sin t_i, y cos t_i + x sin t_i); the
// pairs are elements (i, i + rot / 2) or neighbours (2i, 2i + 1), what lies past rot stays as it is.  Cosines and sines come
// from a table in 32 bits that was made in 64: an angle of a far position has no 32-bit product worth taking.  The products
// are taken in 32 bits and rounded once, to the 16 bits of the cache.
//
// A unit is 16 elements of one head of one row (8 pairs, or 16 elements past rot), two copies of 16 bytes in and out; a
// thread keeps its unit's cosines and sines and walks the heads of a row: K's (rotated), V's (copied), Q's (rotated).
// Bound: the launch and three loads that wait for one another where there are few rows; where there are many HBM, and the same
// loads: a warp looks its row up (sequence, length, page, angles) only when it comes to it, and with 7261 rows nearly every warp of
// the launch has one, so that it hides none of that behind copies of its own.
#include <atomic>

#include "append.cuh"
#include "launch.cuh"
#include "ptx.cuh"

namespace ma {

namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 2;  // heads of a lane in flight together

template <bool BF16>
__device__ __forceinline__ void widen(const uint4& w, float (&x)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2<BF16>(u[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <bool BF16>
__device__ __forceinline__ uint4 narrow(const float (&x)[8]) {
  return make_uint4(pack2<BF16>(x[0], x[1]), pack2<BF16>(x[2], x[3]), pack2<BF16>(x[4], x[5]), pack2<BF16>(x[6], x[7]));
}

// the sequence that row t belongs to: the last whose first row is not behind it (B or more: none)
__device__ __forceinline__ int sequence_of(const AppendArgs& a, int t) {
  int n = 0;
  for (int i = 1 + (threadIdx.x & 31); i <= a.B; i += 32) n += a.cu_q[i] <= t;
  return __reduce_add_sync(0xffffffffu, n);
}

}  // namespace

// kWarps warps take a row together: one where the rows fill the GPU (the three loads of a row's lookups, which wait for one
// another, are then hidden by the other rows of the SM), eight where they do not.  7 prompts of 7261 tokens in all, 32/8 heads of
// 128: 36.7 us = 5.0 TB/s, 0.76 of the copy rate (49 with a CTA to a row); 4 x 8192 tokens, 16/4 heads of 64: 39.9 us = 5.1
// TB/s (89).  Two heads of a lane in flight and three CTAs an SM (4 to 16 bytes spill): 1 and 4 took 37.6 and 40.6 us, 4 and 2
// 34.5 and 41.7, 3 and 3 39.6 and 44.2.  A step of decode (32 rows) takes 2.5 us, a launch and those three loads.
template <bool BF16, int kWarps>
__global__ void __launch_bounds__(kThreads, 3)
append_kernel(const AppendArgs a) {
  constexpr int kGroup = 32 * kWarps, kRowsPerCta = kThreads / kGroup;
  grid_dep_launch();
  grid_dep_wait();
  const int units = a.D / 16;  // of a head
  const int lanes = kGroup / units * units, step = kGroup / units;
  const int tid = threadIdx.x % kGroup;
  const int head0 = div_by(tid, a.by_units), unit = tid - head0 * units;
  const bool turns = a.rope != nullptr && unit * 16 < a.rot;
  const int half = a.rot / 2;
  // the unit's two runs of 8 elements
  const int e0 = turns && !a.interleaved ? unit * 8 : unit * 16;
  const int e1 = turns && !a.interleaved ? half + unit * 8 : unit * 16 + 8;
  const int heads = 2 * a.Hkv + (a.q != nullptr ? a.Hq : 0);

  for (long long row = static_cast<long long>(blockIdx.x) * kRowsPerCta + threadIdx.x / kGroup; row < a.rows;
       row += static_cast<long long>(gridDim.x) * kRowsPerCta) {
    const int t = static_cast<int>(row);
    int b;
    long long first, n_new;
    if (a.cu_q != nullptr) {
      b = sequence_of(a, t);
      if (b >= a.B) continue;  // behind the last sequence's rows
      first = a.cu_q[b];
      n_new = a.cu_q[b + 1] - first;
    } else {
      b = div_by(t, a.by_n);
      first = static_cast<long long>(b) * a.n;
      n_new = a.n;
    }
    const AppendSlot s = append_slot(a, t, first, n_new, a.seq_lens[b],
                                     [&](int i) { return a.table[b * a.table_stride + i]; });
    if (s.bad && tid == 0 && a.status != nullptr) atomicOr(a.status, kErrCache);
    if (s.none || tid >= lanes) continue;
    float cs[8], sn[8];
    const bool turn = turns && s.held;
    if (turn) {
      const float* angles = a.rope + static_cast<long long>(s.pos) * a.rot + unit * 8;
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        *reinterpret_cast<float4*>(cs + i) = *reinterpret_cast<const float4*>(angles + i);
        *reinterpret_cast<float4*>(sn + i) = *reinterpret_cast<const float4*>(angles + half + i);
      }
    }
    const long long seq = a.cu_q != nullptr ? 0 : b, tok = a.cu_q != nullptr ? t : t - first;
    const uint16_t* k = a.k + seq * a.ks[0] + tok * a.ks[2];
    const uint16_t* v = a.v + seq * a.vs[0] + tok * a.vs[2];
    const uint16_t* q = a.q + seq * a.qs[0] + tok * a.qs[2];
    uint16_t* k_to = a.k_cache + s.page * a.kcs[0] + s.at * a.kcs[2];
    uint16_t* v_to = a.v_cache + s.page * a.vcs[0] + s.at * a.vcs[2];
    uint16_t* q_to = a.q_out + seq * a.qos[0] + tok * a.qos[2];
    // K's heads, V's, Q's in a row; kAhead of them in flight together
    for (int h0 = s.held ? head0 : 2 * a.Hkv + head0; h0 < heads; h0 += kAhead * step) {
      uint4 w[kAhead][2];
      uint16_t* to[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int h = h0 + u * step;
        if (h >= heads) break;
        const uint16_t* from;
        if (h < a.Hkv) {
          from = k + h * a.ks[1];
          to[u] = k_to + h * a.kcs[1];
        } else if (h < 2 * a.Hkv) {
          from = v + (h - a.Hkv) * a.vs[1];
          to[u] = v_to + (h - a.Hkv) * a.vcs[1];
        } else {
          from = q + (h - 2 * a.Hkv) * a.qs[1];
          to[u] = q_to + (h - 2 * a.Hkv) * a.qos[1];
        }
        w[u][0] = *reinterpret_cast<const uint4*>(from + e0);
        w[u][1] = *reinterpret_cast<const uint4*>(from + e1);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int h = h0 + u * step;
        if (h >= heads) break;
        if (turn && (h < a.Hkv || h >= 2 * a.Hkv)) {
          float x[8], y[8], p[8], r[8];
          widen<BF16>(w[u][0], x);
          widen<BF16>(w[u][1], y);
          if (a.interleaved) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              p[2 * i] = x[2 * i] * cs[i] - x[2 * i + 1] * sn[i];
              p[2 * i + 1] = x[2 * i + 1] * cs[i] + x[2 * i] * sn[i];
              r[2 * i] = y[2 * i] * cs[4 + i] - y[2 * i + 1] * sn[4 + i];
              r[2 * i + 1] = y[2 * i + 1] * cs[4 + i] + y[2 * i] * sn[4 + i];
            }
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              p[i] = x[i] * cs[i] - y[i] * sn[i];
              r[i] = y[i] * cs[i] + x[i] * sn[i];
            }
          }
          w[u][0] = narrow<BF16>(p);
          w[u][1] = narrow<BF16>(r);
        }
        *reinterpret_cast<uint4*>(to[u] + e0) = w[u][0];
        *reinterpret_cast<uint4*>(to[u] + e1) = w[u][1];
      }
    }
  }
  // A row reports what is wrong with its own sequence; sequences that no row finds by their numbers are looked at here, last, since
  // the stores of the rows take longer to leave than this.
  if (blockIdx.x == 0 && a.cu_q != nullptr && a.status != nullptr)
    for (int b = threadIdx.x; b < a.B; b += kThreads)
      if (append_outside(a, a.cu_q[b], a.cu_q[b + 1], a.seq_lens[b])) atomicOr(a.status, kErrCache);
}

template <bool BF16>
static cudaError_t launch_append_t(const AppendArgs& a, int sms, cudaStream_t st) {
  if (a.rows < sms * 8) return launch_overlapped(append_kernel<BF16, 8>, static_cast<unsigned>(a.rows), kThreads, 0, st, a);
  const int ctas = (a.rows + 7) / 8;
  return launch_overlapped(append_kernel<BF16, 1>, static_cast<unsigned>(ctas < sms * 6 ? ctas : sms * 6), kThreads, 0, st, a);
}

cudaError_t launch_append(bool bf16, const AppendArgs& a, int sms, cudaStream_t st) {
  return bf16 ? launch_append_t<true>(a, sms, st) : launch_append_t<false>(a, sms, st);
}

}  // namespace ma
