// Eviction from a paged cache by accumulated attention weight (gfx950).
//
// Of a sequence's L slots every key head keeps `budget`: the first `sinks`, the
// last `recent`, and of those between the ones with the largest weight sums, of
// equal sums the earlier.  Kept rows go in their order into other pages.
//
// Selection: one work group per (sequence, key head) finds the last kept sum by
// radix selection over the sums' bits in an order that integers compare (NaN
// above all, -0 as 0): 11 bits a pass from the first bit in which any two sums
// differ, so sums of similar size spread over the histogram's bins from its
// first pass on.  A last pass in index order counts what is above the bound, and
// what equals it up to the number that is left to keep.  The sums stay in shared
// memory between the passes where they fit (one read of 4 bytes per slot).
// Copying: 16 bytes a thread; bound by the kept rows read and written.
#include "ca_paged.h"
#include "ca_evict.h"

namespace ca {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBits = 11, kBins = 1 << kBits;
constexpr int kHeld = 24576;  // sums held in shared memory (96 KB)

// Integers in the order of the sums.
__device__ __forceinline__ unsigned sum_key(float x) {
  const unsigned u = __float_as_uint(x + 0.0f);  // -0 becomes 0
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// Sum over the 16 lanes of a row, in each of them.
__device__ __forceinline__ int row_sum(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x128, 0xf, 0xf, true);  // rotations by 8, 4, 2, 1
  x += __builtin_amdgcn_update_dpp(0, x, 0x124, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x122, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x121, 0xf, 0xf, true);
  return x;
}
// Sum of the 16 waves' numbers before wave `wave`.
__device__ __forceinline__ int waves_before(const unsigned* of_wave, int wave) {
  static_assert(kWaves == 16, "one lane row holds the waves' numbers");
  const int l = threadIdx.x & 15;
  return row_sum(l < wave ? (int)of_wave[l] : 0);
}

__global__ __launch_bounds__(kThreads) void ca_evict_select_kernel(EvictIO io) {
  __shared__ unsigned held[kHeld];
  __shared__ int hist[kBins];
  __shared__ unsigned wave_a[kWaves], wave_b[kWaves];
  __shared__ int pick[2];  // bin, sums above it
  const PagedCache& c = io.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = blockIdx.x / c.heads, h = blockIdx.x - b * c.heads;
  const long long room = (long long)c.pages_per_seq * c.div.size;
  int len = c.lengths[b];
  if (len > room) len = (int)room;
  if (len > io.sums_len) len = io.sums_len;
  if (len < 0) len = 0;
  const float* sums = io.sums + (long long)b * io.sums_bs + (long long)h * io.sums_hs;
  const long long out = ((long long)b * c.heads + h) * io.budget;
  int* kept = io.kept + out;
  float* new_sums = io.new_sums + out;
  const int keep = len < io.budget ? len : io.budget;
  if (h == 0 && tid == 0) io.new_lengths[b] = keep;
  for (int i = keep + tid; i < io.budget; i += kThreads) {
    kept[i] = -1;
    new_sums[i] = 0.f;
  }
  if (len <= io.budget) {
    for (int i = tid; i < len; i += kThreads) {
      kept[i] = i;
      new_sums[i] = sums[i];
    }
    return;
  }
  const int lo = io.sinks, hi = len - io.recent;  // the slots that compete, sinks + recent <= budget < len
  int need = io.budget - io.sinks - io.recent;    // of them kept
  unsigned bound = 0xffffffffu;
  if (need > 0) {
    for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
    // the bits all sums share
    unsigned least = 0xffffffffu, most = 0;
    for (int i0 = lo + tid; i0 < hi; i0 += 4 * kThreads) {
      float x[4];  // four loads on their way at a time
#pragma unroll
      for (int q = 0; q < 4; ++q) x[q] = i0 + q * kThreads < hi ? sums[i0 + q * kThreads] : 0.f;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int i = i0 + q * kThreads;
        if (i >= hi) break;
        const unsigned k = sum_key(x[q]);
        if (i - lo < kHeld) held[i - lo] = k;
        least = k < least ? k : least;
        most = k > most ? k : most;
      }
    }
#pragma unroll
    for (int x = 32; x; x >>= 1) {
      const unsigned p = __shfl_xor(least, x), q = __shfl_xor(most, x);
      least = p < least ? p : least;
      most = q > most ? q : most;
    }
    if (lane == 0) {
      wave_a[wave] = least;
      wave_b[wave] = most;
    }
    __syncthreads();
    least = wave_a[lane & 15];
    most = wave_b[lane & 15];
#pragma unroll
    for (int x = 8; x; x >>= 1) {
      const unsigned p = __shfl_xor(least, x), q = __shfl_xor(most, x);
      least = p < least ? p : least;
      most = q > most ? q : most;
    }
    int bits = least == most ? 0 : 32 - __clz(least ^ most);
    unsigned value = bits == 32 ? 0u : most >> bits << bits;  // the bits fixed so far
    while (bits > 0) {
      const int width = bits < kBits ? bits : kBits, shift = bits - width;
      for (int i = lo + tid; i < hi; i += kThreads) {
        const unsigned k = i - lo < kHeld ? held[i - lo] : sum_key(sums[i]);
        if (bits == 32 || (k ^ value) >> bits == 0) atomicAdd(&hist[k >> shift & ((1u << width) - 1)], 1);
      }
      __syncthreads();
      // sums above each bin, from the top: two bins a thread, the top ones first
      const int b0 = kBins - 1 - 2 * tid;
      const int c0 = hist[b0], c1 = hist[b0 - 1];
      hist[b0] = hist[b0 - 1] = 0;  // for the next pass
      int above = c0 + c1;
#pragma unroll
      for (int x = 1; x < 64; x <<= 1) {
        const int y = __shfl_up(above, x);
        if (lane >= x) above += y;
      }
      if (lane == 63) wave_a[wave] = above;
      __syncthreads();
      above += waves_before(wave_a, wave) - c0 - c1;
      // the one bin with fewer than `need` above it and enough with it
      if (above < need && above + c0 >= need) {
        pick[0] = b0;
        pick[1] = above;
      } else if (above + c0 < need && above + c0 + c1 >= need) {
        pick[0] = b0 - 1;
        pick[1] = above + c0;
      }
      __syncthreads();
      value |= (unsigned)pick[0] << shift;
      need -= pick[1];
      bits = shift;
    }
    bound = value;
  }
  // In index order: those above the bound, `need` of those at it.  Each wave
  // takes a run of slots, counts it, and writes it behind what the waves before
  // it hold.
  const int run = (len + 64 * kWaves - 1) / (64 * kWaves) * 64, from = wave * run;
  const int to = from + run < len ? from + run : len;
  auto look = [&](int i, bool& above, bool& equal) {
    above = equal = false;
    if (i >= to) return;
    if (i < lo || i >= hi) {
      above = true;
    } else if (io.budget > io.sinks + io.recent) {
      const unsigned k = i - lo < kHeld ? held[i - lo] : sum_key(sums[i]);
      above = k > bound;
      equal = k == bound;
    }
  };
  int na = 0, ne = 0;
  for (int i = from + lane; i < from + run; i += 64) {
    bool above, equal;
    look(i, above, equal);
    na += __popcll(__ballot(above));
    ne += __popcll(__ballot(equal));
  }
  __syncthreads();  // wave_a and wave_b have been read
  if (lane == 0) {
    wave_a[wave] = na;
    wave_b[wave] = ne;
  }
  __syncthreads();
  na = waves_before(wave_a, wave);
  ne = waves_before(wave_b, wave);
  const unsigned long long before = (1ull << lane) - 1;
  for (int i0 = from + lane; i0 < from + run; i0 += 256) {
    float x[4];  // four loads on their way at a time
#pragma unroll
    for (int q = 0; q < 4; ++q) x[q] = i0 + 64 * q < to ? sums[i0 + 64 * q] : 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int i = i0 + 64 * q;
      bool above, equal;
      look(i, above, equal);
      const unsigned long long ma = __ballot(above), me = __ballot(equal);
      const int a = na + __popcll(ma & before), e = ne + __popcll(me & before);
      if (above || (equal && e < need)) {
        const int at = a + (e < need ? e : need);
        kept[at] = i;
        new_sums[at] = x[q];
      }
      na += __popcll(ma);
      ne += __popcll(me);
    }
  }
}

// Kept rows into their new pages; u counts 16-byte pieces of a (sequence, head).
template <int UNROLL>
__global__ __launch_bounds__(256) void ca_evict_copy_kernel(EvictIO io) {
  const PagedCache& c = io.c;
  const int slices = c.batch * c.heads;
  const int slice = blockIdx.x % slices, part = blockIdx.x / slices, parts = gridDim.x / slices;
  const int b = slice / c.heads, h = slice - b * c.heads;
  const int rows = io.new_lengths[b];
  const int pieces = io.row_pieces;
  const long long total = (long long)rows * pieces;
  const int* kept = io.kept + (long long)slice * io.budget;
  const int* table = c.table + (long long)b * c.table_stride;
  const int* to = io.new_table + (long long)b * io.new_table_stride;
  const char* k = static_cast<const char*>(c.k) + (long long)h * c.head_stride * io.esize;
  const char* v = static_cast<const char*>(c.v) + (long long)h * c.head_stride * io.esize;
  for (long long u0 = (long long)part * 256 * UNROLL; u0 < total; u0 += (long long)parts * 256 * UNROLL) {
    u32x4 kx[UNROLL], vx[UNROLL];
    long long dst[UNROLL];
#pragma unroll
    for (int x = 0; x < UNROLL; ++x) {
      const long long u = u0 + x * 256 + threadIdx.x;
      dst[x] = -1;
      if (u >= total) continue;
      const int row = (int)(u / pieces), piece = (int)(u - (long long)row * pieces);
      const int src = kept[row];
      const int si = page_of(c.div, src), di = page_of(c.div, row);
      const int sp = table[si], dp = to[di];
      if ((unsigned)dp >= (unsigned)c.num_pages) continue;
      dst[x] = ((long long)dp * c.page_stride + (long long)(row - di * (int)c.div.size) * c.row_stride) * io.esize +
               16 * piece;
      kx[x] = vx[x] = u32x4{~0u, ~0u, ~0u, ~0u};  // a page outside the cache: NaN in every type
      if ((unsigned)sp < (unsigned)c.num_pages) {
        const long long at =
            ((long long)sp * c.page_stride + (long long)(src - si * (int)c.div.size) * c.row_stride) * io.esize +
            16 * piece;
        kx[x] = *reinterpret_cast<const u32x4*>(k + at);
        vx[x] = *reinterpret_cast<const u32x4*>(v + at);
      }
    }
#pragma unroll
    for (int x = 0; x < UNROLL; ++x) {
      if (dst[x] < 0) continue;
      *reinterpret_cast<u32x4*>(const_cast<char*>(k) + dst[x]) = kx[x];
      *reinterpret_cast<u32x4*>(const_cast<char*>(v) + dst[x]) = vx[x];
    }
  }
}

}  // namespace

hipError_t launch_evict(const EvictIO& io, hipStream_t s) {
  const int slices = io.c.batch * io.c.heads;
  hipLaunchKernelGGL(ca_evict_select_kernel, dim3((unsigned)slices), dim3(kThreads), 0, s, io);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  constexpr int kUnroll = 4;
  const long long per = 256 * kUnroll;
  long long parts = ((long long)io.budget * io.row_pieces + per - 1) / per;
  const long long most = 16384 / slices > 1 ? 16384 / slices : 1;
  parts = parts < 1 ? 1 : parts > most ? most : parts;
  hipLaunchKernelGGL((ca_evict_copy_kernel<kUnroll>), dim3((unsigned)(slices * parts)), dim3(256), 0, s, io);
  return hipGetLastError();
}

}  // namespace ca
