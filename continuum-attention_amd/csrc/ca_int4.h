// Launch interface of the 4-bit product (ca_int4.hip).
#pragma once
#include "ca_kernels.h"

namespace ca {

struct Int4IO {
  const void* x;         // [M][K], rows x_rs elements apart
  const unsigned* codes;  // [N][row_words], 8 codes a word
  const void* scales;    // [groups][N]
  const void* zeros;     // [groups][N] or null: 8
  void* y;               // [M][N], rows y_rs elements apart
  long long x_rs, y_rs;
  int M, N, K, group, row_words, x_aligned;
};
hipError_t launch_int4(const Int4IO& io, int dtype, hipStream_t s);

}  // namespace ca
