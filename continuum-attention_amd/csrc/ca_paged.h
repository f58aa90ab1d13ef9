// Paged key/value caches: what the attention, append and eviction kernels share.
#pragma once
#include "ca_kernels.h"

namespace ca {

// n / d of n < 2^31 by a product and a shift: with l = ceil(log2 d) and
// m = ceil(2^(31 + l) / d), m d - 2^(31 + l) < d <= 2^l, so that n m / 2^(31 + l)
// exceeds n / d by less than n / 2^31 / d < 1 / d and has the same whole part.
struct PageDiv {
  unsigned mul, shift, size;
};
inline PageDiv page_div(int d) {
  unsigned l = 0;
  while ((1u << l) < (unsigned)d) ++l;
  const unsigned long long one = 1ull << (31 + l);
  return PageDiv{(unsigned)((one + d - 1) / d), 31 + l, (unsigned)d};
}
__host__ __device__ inline int page_of(PageDiv p, int slot) {
  return (int)(((unsigned long long)(unsigned)slot * p.mul) >> p.shift);
}

// A cache as the kernels take it (ca_paged_cache of the public header, with
// strides in elements).
struct PagedCache {
  void *k, *v;
  long long page_stride, head_stride, row_stride;
  const int* table;    // [batch][table_stride]
  const int* lengths;  // [batch], the new tokens included
  const int* starts;   // [batch + 1], first new token of each sequence
  int table_stride, pages_per_seq, num_pages, heads, D, batch;
  PageDiv div;
};

// A sequence's cached length and its new tokens [t0, t0 + n), held to what the
// table and the token tensors have room for whatever the device's numbers say.
struct SeqSpan {
  int len, t0, n;
};
__device__ __forceinline__ SeqSpan seq_span(const PagedCache& c, int b, int tokens) {
  const long long room = (long long)c.pages_per_seq * c.div.size;
  int len = c.lengths[b];
  if (len > room) len = (int)room;
  if (len < 0) len = 0;
  int t0 = c.starts[b], t1 = c.starts[b + 1];
  t0 = t0 < 0 ? 0 : t0 > tokens ? tokens : t0;
  t1 = t1 < t0 ? t0 : t1 > tokens ? tokens : t1;
  return SeqSpan{len, t0, t1 - t0};
}

struct PagedAttnIO {
  PagedCache c;
  const void* q;
  void* out;
  long long q_ts, q_hs, o_ts, o_hs;  // token and head strides, elements
  const float* log_gain;
  float* stats;   // [tokens][heads of q][2]: row shift and 1/Z, or null
  float* part_o;  // [splits][tokens * heads of q][D]
  float* part_ml;  // [splits][tokens * heads of q][2]
  float* sums;    // [batch][heads][sums_rs] weight sums or null
  long long sums_bs, sums_hs;
  int sums_len;
  int tokens, Hq, group;
  int splits, split_keys;  // keys per split (a multiple of a tile's); the last takes the rest
  int row_tiles;           // row tiles of the grid; work groups walk the rest
  // few rows: 2^row_log rows and tile_group tiles of 32 keys share a wave's 16
  // columns; tile_group 0: many rows, on `waves` waves (2, 4, 8) of 16
  int row_log, tile_group, waves, tile_rows;
};
hipError_t launch_paged_attention(const PagedAttnIO& io, int dtype, hipStream_t s);
hipError_t launch_paged_combine(const PagedAttnIO& io, int dtype, hipStream_t s);
hipError_t launch_paged_sums(const PagedAttnIO& io, int dtype, int max_length, hipStream_t s);

}  // namespace ca
