// Products of a few rows with a matrix of 4-bit codes with group scales (gfx950):
//   y[m][n] = sum_k x[m][k] s[n][k / g] (c[n][k] - z[n][k / g]).
//
// Bound by the codes' bytes, K N / 2.  At one instruction a code the vector
// units just keep up with the memory, so a code is never converted: its four
// bits are put into the significand of 16 (fp16: bits 6..9, bf16: bits 3..6),
// which is the number 16 + c exactly, two codes in a shift and an and-or, and the
// matrix cores form sum x (16 + c).  A product with a matrix of ones gives each
// group's sum x, and
//   y += s (sum x (16 + c) - (16 + z) sum x),
// in fp32: the offset is about as large as the codes, so this costs two or three
// bits of the 24.  fp32 x goes through the bf16 form in three exact bf16 limbs.
//
// Tiles.  A wave takes 16 rows n and 128 columns k at a time: lane (i, r) loads
// 16 bytes, the 32 codes k = 32 r .. 32 r + 31 of row i, and gives eight of them to
// each of four 16x16x32 instructions, whose k indexes then stand for
// k = 32 r + 8 j + e; x is read with the same deal.  Groups smaller than 128
// share an instruction, so x is zeroed outside one group at a time.  The waves
// of a work group deal out the columns and add up at the end in a fixed order.
//
// Codes of a word (eight columns): column 2 p in bits 4 p, column 2 p + 1 in bits
// 16 + 4 p, so that a shift by 4 p lines up a pair in the two halves.
#include "ca_int4.h"

namespace ca {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// 16 + c of the pairs of a word, as an operand of eight values.
template <bool BF>
__device__ __forceinline__ u32x4 operand(unsigned w) {
  if constexpr (BF) {
    return u32x4{(w << 3 & 0x00780078u) | 0x41804180u, (w >> 1 & 0x00780078u) | 0x41804180u,
                 (w >> 5 & 0x00780078u) | 0x41804180u, (w >> 9 & 0x00780078u) | 0x41804180u};
  } else {
    return u32x4{(w << 6 & 0x03c003c0u) | 0x4c004c00u, (w << 2 & 0x03c003c0u) | 0x4c004c00u,
                 (w >> 2 & 0x03c003c0u) | 0x4c004c00u, (w >> 6 & 0x03c003c0u) | 0x4c004c00u};
  }
}
template <bool BF>
__device__ __forceinline__ f32x4 product(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (BF)
    return mfma16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c,
                                                  0, 0, 0);
}

// x[m][k .. k + 7] as operand limbs, zeros past K and M.
template <class E, int XL>
__device__ __forceinline__ void load_x(const Int4IO& io, int m, int k, u32x4 (&out)[XL]) {
  const E* p = static_cast<const E*>(io.x) + (long long)m * io.x_rs + k;
  if constexpr (XL == 1) {
    if (m < io.M && io.x_aligned && k + 8 <= io.K) {
      out[0] = *reinterpret_cast<const u32x4*>(p);
      return;
    }
    u32x4 r = {0, 0, 0, 0};
    if (m < io.M) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const unsigned v = k + e < io.K ? reinterpret_cast<const unsigned short*>(p)[e] : 0u;
        r[e >> 1] |= v << (16 * (e & 1));
      }
    }
    out[0] = r;
  } else {
    float v[8];
    const bool fast = m < io.M && io.x_aligned && k + 8 <= io.K;
    if (fast) {
      const f32x4 a = ld4(p), b = ld4(p + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = a[e];
        v[4 + e] = b[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = m < io.M && k + e < io.K ? p[e] : 0.f;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      unsigned h, mm, l;
      split_pair(v[2 * q], v[2 * q + 1], h, mm, l);
      out[0][q] = h;
      out[1][q] = mm;
      out[2][q] = l;
    }
  }
}

constexpr int kMostWaves = 8;

// NT: 16-row tiles of a work group, MT: 16-column (rows of x) tiles, SUB: groups
// in 128 columns (4, 2, 1).
template <class E, int NT, int MT, int SUB>
__global__ __launch_bounds__(64 * kMostWaves) void ca_int4_kernel(Int4IO io) {
  constexpr bool kBf = !std::is_same<E, _Float16>::value;
  constexpr int XL = std::is_same<E, float>::value ? 3 : 1;
  __shared__ float join[kMostWaves][NT * MT][16 * 17];
  const int lane = threadIdx.x & 63, i = lane & 15, r = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), waves = blockDim.x >> 6;
  const int n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16 * MT;
  const u32x4 ones = kBf ? u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u}
                         : u32x4{0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
  const int blocks = (io.K + 127) / 128;
  const int per = SUB == 1 ? io.group / 128 : 1;  // blocks of a group
  f32x4 y[NT][MT];
#pragma unroll
  for (int a = 0; a < NT; ++a)
#pragma unroll
    for (int b = 0; b < MT; ++b) y[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  const unsigned* row[NT];
#pragma unroll
  for (int a = 0; a < NT; ++a) {
    const int n = n0 + 16 * a + i;
    row[a] = io.codes + (long long)(n < io.N ? n : io.N - 1) * io.row_words + 4 * r;
  }
  const E* scales = static_cast<const E*>(io.scales);
  const E* zeros = static_cast<const E*>(io.zeros);
  // a wave takes two neighbouring blocks at a time: 128 bytes of each row
  for (int pair = wave; 2 * pair < blocks; pair += waves) {
    const int first = 2 * pair, count = first + 1 < blocks ? 2 : 1;
    u32x4 w[2][NT];
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int a = 0; a < NT; ++a)
        w[q][a] = q < count ? *reinterpret_cast<const u32x4*>(row[a] + 16 * (first + q)) : u32x4{0, 0, 0, 0};
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      if (q >= count) break;
      const int block = first + q;
      f32x4 acc[SUB][NT][MT], sum[SUB][MT];
#pragma unroll
      for (int s = 0; s < SUB; ++s)
#pragma unroll
        for (int b = 0; b < MT; ++b) {
          sum[s][b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int a = 0; a < NT; ++a) acc[s][a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u32x4 x[MT][XL];
#pragma unroll
        for (int b = 0; b < MT; ++b) load_x<E, XL>(io, m0 + 16 * b + i, 128 * block + 32 * r + 8 * j, x[b]);
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
          const bool in = SUB == 1 || r / (4 / SUB) == s;
#pragma unroll
          for (int b = 0; b < MT; ++b)
#pragma unroll
            for (int l = XL - 1; l >= 0; --l) {
              const u32x4 v = in ? x[b][l] : u32x4{0, 0, 0, 0};
              sum[s][b] = product<kBf>(ones, v, sum[s][b]);
#pragma unroll
              for (int a = 0; a < NT; ++a) acc[s][a][b] = product<kBf>(operand<kBf>(w[q][a][j]), v, acc[s][a][b]);
            }
        }
      }
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
        const int k = 128 * block + 128 / SUB * s;
        if (k >= io.K) break;
        const int g = SUB == 1 ? block / per : SUB * block + s;
#pragma unroll
        for (int a = 0; a < NT; ++a) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int n = n0 + 16 * a + 4 * r + e;
            const long long at = (long long)g * io.N + (n < io.N ? n : io.N - 1);
            const float sc = ld1(scales + at);
            const float off = 16.0f + (zeros ? ld1(zeros + at) : 8.0f);
#pragma unroll
            for (int b = 0; b < MT; ++b) y[a][b][e] = fmaf(sc, fmaf(-off, sum[s][b][e], acc[s][a][b][e]), y[a][b][e]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int a = 0; a < NT; ++a)
#pragma unroll
    for (int b = 0; b < MT; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) join[wave][a * MT + b][(4 * r + e) * 17 + i] = y[a][b][e];
  __syncthreads();
  E* out = static_cast<E*>(io.y);
  for (int u = threadIdx.x; u < 256 * NT * MT; u += blockDim.x) {
    const int n = u % 16, m = u / 16 % 16, tile = u / 256;
    const int nn = n0 + 16 * (tile / MT) + n, mm = m0 + 16 * (tile % MT) + m;
    if (nn >= io.N || mm >= io.M) continue;
    float v = 0.f;
    for (int w = 0; w < waves; ++w) v += join[w][tile][n * 17 + m];
    st1(out + (long long)mm * io.y_rs + nn, v);
  }
}

template <class E, int NT, int MT>
hipError_t run_sub(const Int4IO& io, dim3 grid, dim3 block, hipStream_t s) {
  if (io.group == 32) hipLaunchKernelGGL((ca_int4_kernel<E, NT, MT, 4>), grid, block, 0, s, io);
  else if (io.group == 64) hipLaunchKernelGGL((ca_int4_kernel<E, NT, MT, 2>), grid, block, 0, s, io);
  else hipLaunchKernelGGL((ca_int4_kernel<E, NT, MT, 1>), grid, block, 0, s, io);
  return hipGetLastError();
}
template <class E>
hipError_t run_int4(const Int4IO& io, hipStream_t s) {
  const int pairs = (io.K + 255) / 256;
  const int waves = pairs < kMostWaves ? pairs : kMostWaves;
  const dim3 block(64 * waves);
  const int mt = io.M <= 16 ? 1 : 2;
  const dim3 grid((io.N + 15) / 16, (io.M + 16 * mt - 1) / (16 * mt));
  if (mt == 1) return run_sub<E, 1, 1>(io, grid, block, s);
  return run_sub<E, 1, 2>(io, grid, block, s);
}

}  // namespace

hipError_t launch_int4(const Int4IO& io, int dtype, hipStream_t s) {
  if (dtype == CA_DTYPE_F32) return run_int4<float>(io, s);
  if (dtype == CA_DTYPE_BF16) return run_int4<__bf16>(io, s);
  return run_int4<_Float16>(io, s);
}

}  // namespace ca
