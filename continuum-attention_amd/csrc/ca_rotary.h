// Launch interface of the rotary kernel (ca_rotary.hip).
#pragma once
#include "ca_paged.h"

namespace ca {

struct RotaryIO {
  const void *q, *k, *v;  // v only with a cache
  void *q_out, *k_out;    // k_out only without one
  long long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, qo_ts, qo_hs, ko_ts, ko_hs;  // token, head strides
  const void* positions;
  const double* turns;  // [R / 2] turns per position
  float magnitude;
  int positions64, R, D, Hq, Hk, tokens, half, inverse, aligned16;
  int head_chunks;  // set by the launch
  PagedCache c;     // c.k null: no cache
};
hipError_t launch_rotary(RotaryIO io, int dtype, hipStream_t s);

}  // namespace ca
