// Rotary positions of queries and keys (gfx950): pairs (a, b) of a head's first R
// dims, at position t and with the pair's frequency f (in turns),
//   a' = g (a cos 2 pi f t - b sin 2 pi f t),  b' = g (b cos 2 pi f t + a sin 2 pi f t),
// the other D - R dims as they are; the gradient is the same with -t.  Pairs are
// neighbours (2i, 2i + 1) or halves (i, i + R/2).
//
// Angles.  f t is formed in 64 bits in turns, its whole part dropped there, and
// the fraction, exact to 2^-53 t f, goes to sincospi in 32: an angle of 32 bits
// is off by 2^-24 t f radians, 0.06 at t = 10^6.  The device does 64-bit
// products at half the 32-bit rate, and a thread forms an angle once for all of
// the heads it walks, so the time is that of the bytes.
//
// A thread holds 16 bytes of a head row (two pieces of 16 in the half layout),
// so that a wave reads whole lines; the scalar form takes layouts whose pieces
// do not start on 16 bytes (the multiply-adds are written out, so that both
// round alike).  8192 tokens of 32 heads of 64, bf16: 67 MB each way in 13.2 us,
// 5.1 TB/s, what a copy of a gigabyte reaches.  With a cache the same launch writes
// the rotated keys and the values into their pages: one token's work is three
// launches' latency otherwise.
#include "ca_paged.h"
#include "ca_rotary.h"

namespace ca {

namespace {

template <class E, int N> struct Piece {
  float x[N];
};
template <class E, int N>
__device__ __forceinline__ Piece<E, N> ld_piece(const E* p) {
  Piece<E, N> r;
  if constexpr (N * sizeof(E) == 16) {
    const f32x4 a = ld4(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) r.x[e] = a[e];
    if constexpr (N == 8) {
      const f32x4 b = ld4(p + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) r.x[4 + e] = b[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) r.x[e] = ld1(p + e);
  }
  return r;
}
template <class E, int N>
__device__ __forceinline__ void st_piece(E* p, const Piece<E, N>& r) {
  if constexpr (N * sizeof(E) == 16) {
    st4(p, f32x4{r.x[0], r.x[1], r.x[2], r.x[3]});
    if constexpr (N == 8) st4(p + 4, f32x4{r.x[4], r.x[5], r.x[6], r.x[7]});
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) st1(p + e, r.x[e]);
  }
}

// One thread: unit u of the heads hc, hc + HC, ... of one token.  Units of a
// row: first the rotated ones (interleaved: V elements, V / 2 pairs; halves:
// V elements of each half), then V plain elements each.
template <class E, bool HALF, int V>
__global__ __launch_bounds__(256) void ca_rotary_kernel(RotaryIO io) {
  const int turned = HALF ? io.R / 2 / V : io.R / V;
  const int units = turned + (io.D - io.R) / V;
  const bool cached = io.c.k != nullptr;
  // (more than one turn only where the threads would pass 2^32)
  for (long long id = (long long)blockIdx.x * 256 + threadIdx.x;; id += (long long)gridDim.x * 256) {
    const int u = (int)(id % units);
    const long long rest = id / units;
    const int hc = (int)(rest % io.head_chunks);
    const long long token = rest / io.head_chunks;
    if (token >= io.tokens) return;
    long long cache_row = -1;
    if (cached) {
      int lo = 0, hi = io.c.batch - 1;  // the last sequence that starts at or before the token
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (io.c.starts[mid] <= token) lo = mid; else hi = mid - 1;
      }
      const SeqSpan sp = seq_span(io.c, lo, io.tokens);
      const long long t = token - sp.t0;
      if (t < 0 || t >= sp.n) continue;  // behind the last sequence
      const long long slot = sp.len - sp.n + t;
      if (slot >= 0) {
        const int idx = page_of(io.c.div, (int)slot);
        const int page = io.c.table[(long long)lo * io.c.table_stride + idx];
        if ((unsigned)page < (unsigned)io.c.num_pages)
          cache_row = (long long)page * io.c.page_stride + (slot - (long long)idx * io.c.div.size) * io.c.row_stride;
      }
    }
    constexpr int kPairs = HALF ? V : (V + 1) / 2;
    float cs[kPairs], sn[kPairs];
    const bool turn = u < turned;
    if (turn) {
      const double pos = io.positions64 ? (double)static_cast<const long long*>(io.positions)[token]
                                        : (double)static_cast<const int*>(io.positions)[token];
#pragma unroll
      for (int p = 0; p < kPairs; ++p) {
        const double x = pos * io.turns[u * kPairs + p];
        float s, c;
        sincospif(2.0f * (float)(x - rint(x)), &s, &c);
        cs[p] = c * io.magnitude;
        sn[p] = (io.inverse ? -s : s) * io.magnitude;
      }
    }
    const int d = turn ? u * V : io.R + (u - turned) * V;  // first element (halves: of the first)
    const int heads = io.Hq + io.Hk + (cached ? io.Hk : 0);
    for (int h = hc; h < heads; h += io.head_chunks) {
      const E* src;
      E* dst;
      bool is_v = false;
      if (h < io.Hq) {
        src = static_cast<const E*>(io.q) + token * io.q_ts + (long long)h * io.q_hs;
        dst = static_cast<E*>(io.q_out) + token * io.qo_ts + (long long)h * io.qo_hs;
      } else {
        is_v = h >= io.Hq + io.Hk;
        const int hk = h - io.Hq - (is_v ? io.Hk : 0);
        src = is_v ? static_cast<const E*>(io.v) + token * io.v_ts + (long long)hk * io.v_hs
                   : static_cast<const E*>(io.k) + token * io.k_ts + (long long)hk * io.k_hs;
        if (cached) {
          if (cache_row < 0) continue;
          dst = static_cast<E*>(is_v ? io.c.v : io.c.k) + cache_row + (long long)hk * io.c.head_stride;
        } else {
          dst = static_cast<E*>(io.k_out) + token * io.ko_ts + (long long)hk * io.ko_hs;
        }
      }
      Piece<E, V> a = ld_piece<E, V>(src + d);
      if constexpr (HALF) {
        if (turn) {
          Piece<E, V> b = ld_piece<E, V>(src + d + io.R / 2);
          if (!is_v) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const float x = a.x[e], y = b.x[e];
              a.x[e] = fmaf(x, cs[e], -(y * sn[e]));
              b.x[e] = fmaf(y, cs[e], x * sn[e]);
            }
          }
          st_piece<E, V>(dst + d + io.R / 2, b);
        }
      } else {
        if (turn && !is_v) {
#pragma unroll
          for (int e = 0; e < V / 2; ++e) {
            const float x = a.x[2 * e], y = a.x[2 * e + 1];
            a.x[2 * e] = fmaf(x, cs[e], -(y * sn[e]));
            a.x[2 * e + 1] = fmaf(y, cs[e], x * sn[e]);
          }
        }
      }
      st_piece<E, V>(dst + d, a);
    }
  }
}

template <class E>
hipError_t run_rotary(RotaryIO& io, hipStream_t s) {
  constexpr int kWide = 16 / sizeof(E);
  const bool wide = io.aligned16 && io.D % kWide == 0 && (io.half ? io.R / 2 : io.R) % kWide == 0;
  const int V = wide ? kWide : io.half ? 1 : 2;
  const int units = (io.half ? io.R / 2 : io.R) / V + (io.D - io.R) / V;
  const int heads = io.Hq + io.Hk * (io.c.k ? 2 : 1);
  // heads a thread walks with one set of angles: up to 8, as long as 2^18
  // threads (1024 on each CU) remain
  long long per = (long long)io.tokens * heads * units >> 18;
  per = per < 1 ? 1 : per > 8 ? 8 : per;
  io.head_chunks = (int)((heads + per - 1) / per);
  const long long blocks = ((long long)io.tokens * io.head_chunks * units + 255) / 256;
  const dim3 grid((unsigned)(blocks < 1 << 23 ? blocks : 1 << 23)), block(256);
  if (io.half) {
    if (wide) hipLaunchKernelGGL((ca_rotary_kernel<E, true, kWide>), grid, block, 0, s, io);
    else hipLaunchKernelGGL((ca_rotary_kernel<E, true, 1>), grid, block, 0, s, io);
  } else {
    if (wide) hipLaunchKernelGGL((ca_rotary_kernel<E, false, kWide>), grid, block, 0, s, io);
    else hipLaunchKernelGGL((ca_rotary_kernel<E, false, 2>), grid, block, 0, s, io);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_rotary(RotaryIO io, int dtype, hipStream_t s) {
  if (dtype == CA_DTYPE_F32) return run_rotary<float>(io, s);
  if (dtype == CA_DTYPE_BF16) return run_rotary<__bf16>(io, s);
  return run_rotary<_Float16>(io, s);
}

}  // namespace ca
