// New tokens into a paged cache, rotated by their positions on the way.
//
// With the angle t_i = pos * theta^(-2i / rot) of pair i, (x, y) becomes (x cos t_i - y sin t_i, y cos t_i + x sin t_i); the
// pairs are elements (i, i + rot / 2) or neighbours (2i, 2i + 1), what lies past rot stays as it is.  Cosines and sines come
// from a table in 32 bits that was made in 64: an angle of a far position has no 32-bit product worth taking.  The products
// are taken in 32 bits and rounded once, to the 16 bits of the cache.
//
// A unit is 16 elements of one head of one row (8 pairs, or 16 elements past rot), two copies of 16 bytes in and out; a
// thread keeps its unit's cosines and sines and walks the heads of a row: K's (rotated), V's (copied), Q's (rotated).
// Bound: HBM where there are many rows, the launch and three loads that wait for one another where there are few.
#include <atomic>

#include "append.cuh"
#include "launch.cuh"
#include "ptx.cuh"

namespace ma {

namespace {

constexpr int kThreads = 256;

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

template <bool BF16>
__global__ void __launch_bounds__(kThreads)
append_kernel(const AppendArgs a) {
  grid_dep_launch();
  grid_dep_wait();
  const int units = a.D / 16;  // of a head
  const int lanes = kThreads / units * units;
  const int tid = threadIdx.x;
  const int unit = tid - div_by(tid, a.by_units) * units, lane0 = div_by(tid, a.by_units), step = lanes / units;
  const bool turns = a.rope != nullptr && unit * 16 < a.rot;
  const int half = a.rot / 2;
  // the unit's two runs of 8 elements
  const int e0 = turns && !a.interleaved ? unit * 8 : unit * 16;
  const int e1 = turns && !a.interleaved ? half + unit * 8 : unit * 16 + 8;
  const int heads = 2 * a.Hkv + (a.q != nullptr ? a.Hq : 0);

  for (int t = blockIdx.x; t < a.rows; t += gridDim.x) {
    int b;
    long long first, n_new;
    if (a.cu_q != nullptr) {
      b = sequence_of(a, t);
      if (b >= a.B) continue;  // rows behind the last sequence are left as they are
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
    if (tid >= lanes) continue;
    float cs[8], sn[8];
    const bool turn = turns && s.held;
    if (turn) {
      const float* row = a.rope + static_cast<long long>(s.pos) * a.rot + unit * 8;
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        *reinterpret_cast<float4*>(cs + i) = *reinterpret_cast<const float4*>(row + i);
        *reinterpret_cast<float4*>(sn + i) = *reinterpret_cast<const float4*>(row + half + i);
      }
    }
    const long long seq = a.cu_q != nullptr ? 0 : b, tok = a.cu_q != nullptr ? t : t - first;
    for (int h = lane0; h < heads; h += step) {
      const uint16_t* src;
      uint16_t* dst;
      bool rotate = turn;
      if (h < 2 * a.Hkv) {
        if (!s.held) continue;
        const int hk = h < a.Hkv ? h : h - a.Hkv;
        if (h < a.Hkv) {
          src = a.k + seq * a.ks[0] + hk * a.ks[1] + tok * a.ks[2];
          dst = a.k_cache + s.page * a.kcs[0] + hk * a.kcs[1] + s.at * a.kcs[2];
        } else {
          src = a.v + seq * a.vs[0] + hk * a.vs[1] + tok * a.vs[2];
          dst = a.v_cache + s.page * a.vcs[0] + hk * a.vcs[1] + s.at * a.vcs[2];
          rotate = false;
        }
      } else {
        const int hq = h - 2 * a.Hkv;
        src = a.q + seq * a.qs[0] + hq * a.qs[1] + tok * a.qs[2];
        dst = a.q_out + seq * a.qos[0] + hq * a.qos[1] + tok * a.qos[2];
      }
      uint4 w0 = *reinterpret_cast<const uint4*>(src + e0), w1 = *reinterpret_cast<const uint4*>(src + e1);
      if (rotate) {
        float x[8], y[8], u[8], w[8];
        widen<BF16>(w0, x);
        widen<BF16>(w1, y);
        if (a.interleaved) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            u[2 * i] = x[2 * i] * cs[i] - x[2 * i + 1] * sn[i];
            u[2 * i + 1] = x[2 * i + 1] * cs[i] + x[2 * i] * sn[i];
            w[2 * i] = y[2 * i] * cs[4 + i] - y[2 * i + 1] * sn[4 + i];
            w[2 * i + 1] = y[2 * i + 1] * cs[4 + i] + y[2 * i] * sn[4 + i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            u[i] = x[i] * cs[i] - y[i] * sn[i];
            w[i] = y[i] * cs[i] + x[i] * sn[i];
          }
        }
        w0 = narrow<BF16>(u);
        w1 = narrow<BF16>(w);
      }
      *reinterpret_cast<uint4*>(dst + e0) = w0;
      *reinterpret_cast<uint4*>(dst + e1) = w1;
    }
  }
}

cudaError_t launch_append(bool bf16, const AppendArgs& a, int sms, cudaStream_t st) {
  const unsigned grid = static_cast<unsigned>(a.rows < sms * 8 ? a.rows : sms * 8);
  return bf16 ? launch_overlapped(append_kernel<true>, grid, kThreads, 0, st, a)
              : launch_overlapped(append_kernel<false>, grid, kThreads, 0, st, a);
}

}  // namespace ma
