// Launch interface of the 4-bit product (ca_int4.hip).
#pragma once
#include "ca_kernels.h"

namespace ca {

struct Int4IO {
  const void* x;         // [M][K], rows x_rs elements apart
  const unsigned* codes;  // [N / 16, K / 128, rounded up][64 lanes][4 words]
  const void* scales;    // [groups][N, to a multiple of 16]
  const void* zeros;     // the same, or null: 8
  void* y;               // [M][N], rows y_rs elements apart
  long long x_rs, y_rs;
  int M, N, K, group, x_aligned;
};
hipError_t launch_int4(const Int4IO& io, int dtype, hipStream_t s);

}  // namespace ca
