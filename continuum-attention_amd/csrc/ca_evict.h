// Launch interface of the eviction kernels (ca_evict.hip).
#pragma once
#include "ca_paged.h"

namespace ca {

struct EvictIO {
  PagedCache c;
  const float* sums;  // [batch][heads][sums_len]
  long long sums_bs, sums_hs;
  int sums_len, budget, sinks, recent;
  const int* new_table;  // [batch][new_table_stride]
  long long new_table_stride;
  int* kept;         // [batch][heads][budget], -1 behind the last kept
  float* new_sums;   // [batch][heads][budget], 0 behind the last kept
  int* new_lengths;  // [batch]
  int row_pieces, esize;  // 16-byte pieces of a row, bytes of an element
  int parts;  // work groups per (sequence, head); set by the launch
};
hipError_t launch_evict(EvictIO io, hipStream_t s);

}  // namespace ca
