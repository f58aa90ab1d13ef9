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
// bits of the 24, which 16-bit results do not show.  fp32 x goes through the bf16
// form in three exact bf16 limbs, and there c - z is formed as it is (six
// instructions a pair instead of two), so that fp32 results keep those bits
// (error 5.9e-7 -> 1.2e-7, a plain fp32 product's 1.1e-7).
//
// Tiles.  A wave takes 16 rows n and 128 columns k at a time, stored as the 1 KB that
// it reads with one load: lane (i, r) gets the codes of row i, columns
// 32 j + 8 r + e, j = 0..3, e = 0..7, eight for each of four 16x16x32 instructions, so
// that one instruction covers 32 neighbouring columns and no group is split by
// one.  (Row by row, a load touched 16 lines, and the address unit bounded it:
// [16,8192] x [8192,8192] 26 us.)  x passes through shared memory for the same
// reason: read as 256 bytes of a row by 16 lanes, handed over as operands.  Each
// group's sums are scaled where they end.  The waves of a work group deal out the
// columns and add up at the end in a fixed order.  A wave loads a block, multiplies
// it, loads the next: other waves hide its loads.  (Two blocks a wave in flight
// and half as many waves: [16,8192] x [8192,8192], groups of 64, 14.0 us against
// 12.0, which is 2.9 TB/s of codes; codes alone loaded ahead: 12.9.)
//
// Codes of a word (eight columns): column 2 p in bits 4 p, column 2 p + 1 in bits
// 16 + 4 p, so that a shift by 4 p lines up a pair in the two halves.  Rows of
// codes, and of scales and zero points ([group][row]), are padded to 16.
#include "ca_int4.h"

#include <algorithm>

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
// c - z of the pairs of a word, off = 16 + z (whole numbers below 2^8: exact).
__device__ __forceinline__ u32x4 operand_less(unsigned w, float off) {
  u32x4 r = operand<true>(w);
#pragma unroll
  for (int p = 0; p < 4; ++p)
    r[p] = cvt_pk_bf16(__uint_as_float(r[p] << 16) - off, __uint_as_float(r[p] & 0xffff0000u) - off);
  return r;
}
template <bool BF>
__device__ __forceinline__ f32x4 product(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (BF)
    return mfma16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c,
                                                  0, 0, 0);
}

// 16 bytes of a row of x at p, `left` columns before its end, element by element.
template <class E>
__device__ __forceinline__ u32x4 load_part(const E* p, int left) {
  constexpr int kVec = 16 / sizeof(E);
  u32x4 r = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < kVec; ++e) {
    if (e >= left) break;
    if constexpr (kVec == 8) r[e >> 1] |= (unsigned)reinterpret_cast<const unsigned short*>(p)[e] << (16 * (e & 1));
    else r[e] = reinterpret_cast<const unsigned*>(p)[e];
  }
  return r;
}
// Eight values as operand limbs (16-bit values are their own).
template <class E, int XL>
__device__ __forceinline__ void operand_x(const E* p, u32x4 (&out)[XL]) {
  if constexpr (XL == 1) {
    out[0] = *reinterpret_cast<const u32x4*>(p);
  } else {
    const f32x4 a = ld4(p), b = ld4(p + 4);
    const float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      unsigned h, m, l;
      split_pair(v[2 * q], v[2 * q + 1], h, m, l);
      out[0][q] = h;
      out[1][q] = m;
      out[2][q] = l;
    }
  }
}

// NT: 16-row tiles of a work group, MT: 16-column (rows of x) tiles, SUB: groups
// in 128 columns (4, 2, 1), WAVES: the most of a work group.
template <class E, int NT, int MT, int SUB, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void ca_int4_kernel(Int4IO io) {
  constexpr bool kBf = !std::is_same<E, _Float16>::value;
  constexpr int XL = std::is_same<E, float>::value ? 3 : 1;
  constexpr int kPer = 4 / SUB;  // instructions of a group
  constexpr bool kF32 = XL == 3;
  constexpr int kVec = 16 / sizeof(E), kPieces = 128 / kVec;  // 16-byte pieces of a row's 128 columns
  constexpr int kLoads = 16 * MT * kPieces / 64;              // of x per lane and block
  constexpr int kXRow = 128 + kVec;                           // staged row: 16 bytes of padding
  constexpr int kXBytes = 16 * MT * kXRow * (int)sizeof(E), kJoinBytes = NT * MT * 16 * 17 * 4;
  __shared__ __attribute__((aligned(16))) unsigned char lds[WAVES][kXBytes > kJoinBytes ? kXBytes : kJoinBytes];
  const int lane = threadIdx.x & 63, i = lane & 15, r = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), waves = blockDim.x >> 6;
  const int n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16 * MT;
  const u32x4 ones = kBf ? u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u}
                         : u32x4{0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
  const int blocks = (io.K + 127) / 128, rows = (io.N + 15) / 16 * 16;
  const int per = SUB == 1 ? io.group / 128 : 1;  // blocks of a group
  const int groups = (io.K + io.group - 1) / io.group;
  f32x4 y[NT][MT];
#pragma unroll
  for (int a = 0; a < NT; ++a)
#pragma unroll
    for (int b = 0; b < MT; ++b) y[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  // (a work group's last tiles may lie behind the padded rows: their loads
  // take the first tile's place and nothing of them is written)
  int n[NT];
  const unsigned* row[NT];
#pragma unroll
  for (int a = 0; a < NT; ++a) {
    n[a] = n0 + 16 * a < rows ? n0 + 16 * a : n0;
    row[a] = io.codes + (long long)(n[a] / 16) * blocks * 256 + 4 * lane;
  }
  const E* x_row[kLoads];  // this lane's pieces of x
#pragma unroll
  for (int q = 0; q < kLoads; ++q) {
    const int m = m0 + (lane + 64 * q) / kPieces;
    x_row[q] = m < io.M ? static_cast<const E*>(io.x) + (long long)m * io.x_rs + lane % kPieces * kVec : nullptr;
  }
  // What a block of 128 columns needs.
  struct Block {
    u32x4 codes[NT], x[kLoads];
    typename Raw4<E>::type scale[SUB][NT], zero[SUB][NT];
    float row_zero[SUB][NT];  // fp32: of the row whose codes this lane holds
  };
  auto load = [&](int block, Block& o) {
#pragma unroll
    for (int a = 0; a < NT; ++a) o.codes[a] = *reinterpret_cast<const u32x4*>(row[a] + 256 * (long long)block);
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      int g = SUB == 1 ? block / per : SUB * block + s;
      if (SUB > 1 && g >= groups) g = groups - 1;  // columns past K: x is zero there
#pragma unroll
      for (int a = 0; a < NT; ++a) {
        const long long at = (long long)g * rows + n[a] + 4 * r;
        o.scale[s][a] = ld_raw4(static_cast<const E*>(io.scales) + at);
        if constexpr (kF32)
          o.row_zero[s][a] = io.zeros ? static_cast<const float*>(io.zeros)[(long long)g * rows + n[a] + i] : 8.f;
        else if (io.zeros)
          o.zero[s][a] = ld_raw4(static_cast<const E*>(io.zeros) + at);
      }
    }
    // rows past M are zero; whole aligned blocks are the rule
    if (io.x_aligned && 128 * block + 128 <= io.K) {
#pragma unroll
      for (int q = 0; q < kLoads; ++q)
        o.x[q] = x_row[q] ? *reinterpret_cast<const u32x4*>(x_row[q] + 128 * block) : u32x4{0, 0, 0, 0};
    } else {
#pragma unroll
      for (int q = 0; q < kLoads; ++q)
        o.x[q] = x_row[q] ? load_part<E>(x_row[q] + 128 * block, io.K - 128 * block - lane % kPieces * kVec)
                          : u32x4{0, 0, 0, 0};
    }
  };
  E* xs = reinterpret_cast<E*>(lds[wave]);
  auto add = [&](const Block& o) {
    wave_lds_sync();  // the block before has been read
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      const int at = lane + 64 * q;
      *reinterpret_cast<u32x4*>(xs + at / kPieces * kXRow + at % kPieces * kVec) = o.x[q];
    }
    wave_lds_sync();
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      f32x4 sum[MT], acc[NT][MT];
#pragma unroll
      for (int b = 0; b < MT; ++b) {
        sum[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int a = 0; a < NT; ++a) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int j = kPer * s; j < kPer * s + kPer; ++j) {
        u32x4 c[NT];
#pragma unroll
        for (int a = 0; a < NT; ++a) {
          if constexpr (kF32) c[a] = operand_less(o.codes[a][j], 16.0f + o.row_zero[s][a]);
          else c[a] = operand<kBf>(o.codes[a][j]);
        }
#pragma unroll
        for (int b = 0; b < MT; ++b) {
          u32x4 x[XL];
          operand_x<E, XL>(xs + (16 * b + i) * kXRow + 32 * j + 8 * r, x);
#pragma unroll
          for (int l = XL - 1; l >= 0; --l) {
            if (!kF32) sum[b] = product<kBf>(ones, x[l], sum[b]);
#pragma unroll
            for (int a = 0; a < NT; ++a) acc[a][b] = product<kBf>(c[a], x[l], acc[a][b]);
          }
        }
      }
#pragma unroll
      for (int a = 0; a < NT; ++a) {
        const f32x4 sc = raw_to_f32(o.scale[s][a], (const E*)nullptr);
        f32x4 off = f32x4{24.f, 24.f, 24.f, 24.f};
        if (!kF32 && io.zeros) off = raw_to_f32(o.zero[s][a], (const E*)nullptr) + 16.0f;
#pragma unroll
        for (int b = 0; b < MT; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e) y[a][b][e] = fmaf(sc[e], kF32 ? acc[a][b][e] : fmaf(-off[e], sum[b][e], acc[a][b][e]), y[a][b][e]);
      }
    }
  };
  auto block_of = [&](int k) { return wave + waves * k; };
  Block p;
  for (int k = 0; block_of(k) < blocks; ++k) {
    load(block_of(k), p);
    add(p);
  }
  wave_lds_sync();
  float* join = reinterpret_cast<float*>(lds[wave]);
#pragma unroll
  for (int a = 0; a < NT; ++a)
#pragma unroll
    for (int b = 0; b < MT; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) join[(a * MT + b) * 272 + (4 * r + e) * 17 + i] = y[a][b][e];
  __syncthreads();
  E* out = static_cast<E*>(io.y);
  for (int u = threadIdx.x; u < 256 * NT * MT; u += blockDim.x) {
    const int nn = u % 16, m = u / 16 % 16, tile = u / 256;
    const int nr = n0 + 16 * (tile / MT) + nn, mr = m0 + 16 * (tile % MT) + m;
    if (nr >= io.N || mr >= io.M) continue;
    float v = 0.f;
    for (int q = 0; q < waves; ++q) v += reinterpret_cast<const float*>(lds[q])[tile * 272 + nn * 17 + m];
    st1(out + (long long)mr * io.y_rs + nr, v);
  }
}

template <class E, int NT, int MT>
hipError_t run_sub(const Int4IO& io, dim3 grid, hipStream_t s) {
  const int blocks = (io.K + 127) / 128;
  auto launch = [&](auto kernel, int most) {
    hipLaunchKernelGGL(kernel, grid, dim3(64 * std::min(blocks, most)), 0, s, io);
  };
  // 16 waves where there is a work group for each CU at most, unless groups of 32
  // take too many registers; with more work groups eight are faster (us with 16 /
  // 8: [64,1024] x [4096,1024] bf16 6.5 / 5.0, [256,4096] x [4096,4096] 46 / 38)
  const bool few = (long long)grid.x * grid.y <= 256;
  if (io.group == 32) {
    if constexpr (NT == 2) return hipErrorInvalidValue;  // (not asked for)
    else launch(ca_int4_kernel<E, NT, MT, 4, 8>, 8);
  } else if (io.group == 64 && few) launch(ca_int4_kernel<E, NT, MT, 2, 16>, 16);
  else if (io.group == 64) launch(ca_int4_kernel<E, NT, MT, 2, 8>, 8);
  else if (few) launch(ca_int4_kernel<E, NT, MT, 1, 16>, 16);
  else launch(ca_int4_kernel<E, NT, MT, 1, 8>, 8);
  return hipGetLastError();
}
template <class E>
hipError_t run_int4(const Int4IO& io, hipStream_t s) {
  // fp32 rows take twice the shared memory: 16 at a time
  const int mt = io.M <= 16 || sizeof(E) == 4 ? 1 : 2;
  const unsigned my = (io.M + 16 * mt - 1) / (16 * mt);
  const int tiles = (io.N + 15) / 16;
  if constexpr (sizeof(E) == 2) {
    if (mt == 2) return run_sub<E, 1, 2>(io, dim3(tiles, my), s);
    // two tiles share x where that still leaves a work group for each of 256 CUs, and
    // groups of 32, which take the registers, stay with one ([16,8192] x [8192,8192],
    // us with one / two, groups of 32: 16.7 / 17.5, of 64: 13.9 / 12.0, of 128: 13.2 /
    // 11.1; [1,1024] x [4096,1024] 3.6 / 4.2)
    if (tiles >= 512 && io.group > 32) return run_sub<E, 2, 1>(io, dim3((tiles + 1) / 2, my), s);
  }
  return run_sub<E, 1, 1>(io, dim3(tiles, my), s);
}

}  // namespace

hipError_t launch_int4(const Int4IO& io, int dtype, hipStream_t s) {
  if (dtype == CA_DTYPE_F32) return run_int4<float>(io, s);
  if (dtype == CA_DTYPE_BF16) return run_int4<__bf16>(io, s);
  return run_int4<_Float16>(io, s);
}

}  // namespace ca
