// Eviction from a paged cache by accumulated attention weight (gfx950).
//
// Of a sequence's L slots every key head keeps `budget`: the first `sinks`, the
// last `recent`, and of those between the ones with the largest weight sums, of
// equal sums the earlier.  Kept rows go in their order into other pages.
//
// Selection: a work group finds the last kept sum of a (sequence, key head) by radix
// selection over the sums' bits in an order that integers compare (NaN above all,
// -0 as 0): 11 bits a pass from the first bit in which any two sums differ, so sums
// of similar size spread over the histogram's bins from its first pass on.  The
// sums stay in shared memory between the passes where they fit (one read of 4
// bytes per slot).  Then its waves go through runs of slots in order: a wave
// counts what is above the bound, and what equals it up to the number left to
// keep, writes the numbers and copies the rows, 16 bytes a lane, as it finds
// them.  With few (sequence, head)s several work groups select alike and share the
// copying by chunks of 64 slots.  128 rows of 8192 sums, up to a quarter kept (64
// columns of bf16): 32 us with four work groups a row, 36 with two; a copy kernel
// of its own behind the selection took 17 + 17 us and the gap between the two.
#include "ca_paged.h"
#include "ca_evict.h"

namespace ca {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBits = 11, kBins = 1 << kBits;
constexpr int kHeld = 16384;  // sums held in shared memory (64 KB: two work groups fit a CU)

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

// Rows from[0 .. count) to new slots first, first + 1, ..., by one wave.
__device__ __forceinline__ void copy_rows(const PagedCache& c, const int* table, const int* new_table, char* k,
                                          char* v, const EvictIO& io, const int* from, int first, int count) {
  const int total = count * io.row_pieces;
  for (int u0 = threadIdx.x & 63; u0 < total; u0 += 128) {
    u32x4 kx[2], vx[2];
    long long to[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int u = u0 + 64 * q;
      to[q] = -1;
      if (u >= total) continue;
      const int row = u / io.row_pieces, piece = u - row * io.row_pieces;
      const int src = from[row], dst = first + row;
      const int si = page_of(c.div, src), di = page_of(c.div, dst);
      const int sp = table[si], dp = new_table[di];
      if ((unsigned)dp < (unsigned)c.num_pages)
        to[q] = ((long long)dp * c.page_stride + (long long)(dst - di * (int)c.div.size) * c.row_stride) * io.esize +
                16 * piece;
      kx[q] = vx[q] = u32x4{~0u, ~0u, ~0u, ~0u};  // a page outside the cache: NaN in every type
      if ((unsigned)sp < (unsigned)c.num_pages) {
        const long long at =
            ((long long)sp * c.page_stride + (long long)(src - si * (int)c.div.size) * c.row_stride) * io.esize +
            16 * piece;
        kx[q] = *reinterpret_cast<const u32x4*>(k + at);
        vx[q] = *reinterpret_cast<const u32x4*>(v + at);
      }
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      if (to[q] < 0) continue;
      *reinterpret_cast<u32x4*>(k + to[q]) = kx[q];
      *reinterpret_cast<u32x4*>(v + to[q]) = vx[q];
    }
  }
}

__global__ __launch_bounds__(kThreads) void ca_evict_kernel(EvictIO io) {
  __shared__ unsigned held[kHeld];
  __shared__ int hist[kBins];
  __shared__ unsigned wave_a[kWaves], wave_b[kWaves];
  __shared__ int pick[2];  // bin, sums above it
  __shared__ int found[kWaves][64];
  const PagedCache& c = io.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int slice = blockIdx.x / io.parts, part = blockIdx.x - slice * io.parts;
  const int b = slice / c.heads, h = slice - b * c.heads;
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
  if (part == 0) {
    if (h == 0 && tid == 0) io.new_lengths[b] = keep;
    for (int i = keep + tid; i < io.budget; i += kThreads) {
      kept[i] = -1;
      new_sums[i] = 0.f;
    }
  }
  const bool all = len <= io.budget;
  const int lo = io.sinks, hi = len - io.recent;  // the slots that compete, sinks + recent <= budget < len
  int need = all ? 0 : io.budget - io.sinks - io.recent;  // of them kept
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
    if (all || i < lo || i >= hi) {
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
  const int* table = c.table + (long long)b * c.table_stride;
  const int* new_table = io.new_table + (long long)b * io.new_table_stride;
  char* k = static_cast<char*>(c.k) + (long long)h * c.head_stride * io.esize;
  char* v = static_cast<char*>(c.v) + (long long)h * c.head_stride * io.esize;
  int* mine = found[wave];
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
      const int first = na + (ne < need ? ne : need);  // new slot of the chunk's first
      const bool take = above || (equal && ne + __popcll(me & before) < need);
      na += __popcll(ma);
      ne += __popcll(me);
      if ((i - lane) / 64 % io.parts != part) continue;  // (the same for the wave)
      const unsigned long long taken = __ballot(take);
      const int count = __popcll(taken);
      if (take) {
        const int at = __popcll(taken & before);
        kept[first + at] = i;
        new_sums[first + at] = x[q];
        mine[at] = i;
      }
      wave_lds_sync();
      copy_rows(c, table, new_table, k, v, io, mine, first, count);
      wave_lds_sync();
    }
  }
}

}  // namespace

hipError_t launch_evict(EvictIO io, hipStream_t s) {
  const int slices = io.c.batch * io.c.heads;
  // two work groups fit each of 256 CUs
  io.parts = slices >= 512 ? 1 : slices > 64 ? 512 / slices : 8;
  hipLaunchKernelGGL(ca_evict_kernel, dim3((unsigned)(slices * io.parts)), dim3(kThreads), 0, s, io);
  return hipGetLastError();
}

}  // namespace ca
