// Continuum Attention of new tokens over a paged key/value cache (gfx950).
//
// A sequence of cached length L (its n new tokens included) has its query t at
// slot p = L - n + t, which sees keys 0..p with the operator's weights: the
// scores are linear between neighbouring slots, each key takes the integral of
// e^score against its hat function, keys 0 and p half a token more (segment
// math in ca_common.h).  The rows of one key head are its new tokens times the
// query heads that share it, r = t * group + g.
//
// Products on 16x16 matrix instructions, 16 rows by 32 keys at a time.  S^T = K Q^T:
// the keys' rows are dealt so that lane row G = lane / 16 holds slots 8G .. 8G + 7
// of query lane % 16; 16-bit K comes straight from memory into operand registers
// (a row's D values are dealt to the four lane rows in quarters, the queries'
// alike, so that a lane reads consecutive bytes).  O^T += V^T W^T takes the lane's
// own weights as the other operand; V passes through shared memory, where it is
// read transposed.  16-bit operands are exact in the 16-bit instructions; the
// weights go as two 16-bit limbs (relative error 2^-17 in bf16, 2^-20 in fp16,
// against half a step of 2^-9 and 2^-12 that the output's rounding makes).
//
// Three kernels walk the keys: many rows (ca_paged_attention_kernel, bound by the
// segments' vector instructions), few rows (ca_paged_few_kernel: up to 8 per key
// head, fp32 16, single tokens above all; bound by the bytes of K and V), and the
// weight sums (ca_paged_sums_kernel).  Keys are cut between work groups where the
// rows alone do not fill the device, and joined by ca_paged_combine_kernel.
#include "ca_paged.h"

#include <algorithm>

namespace ca {

namespace {

constexpr int kOwned = 30;  // keys that a tile of the weight sums owns

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma16_f16(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16_f32(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16_of(u32x4 a, u32x4 b, f32x4 c, const __bf16*) {
  return mfma16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c);
}
__device__ __forceinline__ f32x4 mfma16_of(u32x4 a, u32x4 b, f32x4 c, const _Float16*) {
  return mfma16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c);
}

__device__ __forceinline__ float lane_xor16(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return (threadIdx.x & 16) ? __uint_as_float(r[0]) : __uint_as_float(r[1]);
}
// Value of the same lane in the lane row before (row 0: row 3's) and behind.
__device__ __forceinline__ float row_before(float x) {
  const float a = lane_xor16(x), b = lane_xor16(xhalf(x));
  return (threadIdx.x & 16) ? a : b;
}
__device__ __forceinline__ float row_behind(float x) {
  const float a = lane_xor16(x), b = lane_xor16(xhalf(x));
  return (threadIdx.x & 16) ? b : a;
}
// Value of the lane N places on in the 16 lanes of a row, around its end.
template <int N>
__device__ __forceinline__ float row_rotated(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 + N, 0xf, 0xf, true));
}
__device__ __forceinline__ float rows_max(float x) {
  x = fmaxf(x, lane_xor16(x));
  return fmaxf(x, xhalf(x));
}
__device__ __forceinline__ float rows_sum(float x) {
  x += lane_xor16(x);
  return x + xhalf(x);
}

// The weights of fp16 values go into fp16 limbs, whose range ends at 65504: with
// scores at most 2^8 above the row's shift (kLazyRescale) a weight is below
// 2.5 * 2^8, and 2^6 times that still fits; below, what 16-bit limbs lose is
// under 2^-31 of the row's largest weight.  The factor stays in Z and O.
template <class E> constexpr float weight_octaves() {
  return std::is_same<E, _Float16>::value ? 6.0f : 0.0f;
}

template <class E, int DT> struct Tile {
  static constexpr bool kF32 = std::is_same<E, float>::value;
  static constexpr int kVec = kF32 ? 4 : 8;          // elements in 16 bytes
  static constexpr int kPieces = DT / 4 / kVec;      // 16-byte pieces of a lane's quarter row
  static constexpr int kRow = DT + (kF32 ? 4 : 16);  // elements of a V row in shared memory
  static constexpr int kChunks = DT / kVec;          // 16-byte chunks of a row
};

// Rows of 16 queries (one per lane % 16) and their operands.
template <class E, int DT> struct Rows {
  u32x4 q[Tile<E, DT>::kPieces];
  int pos;        // the query's slot; -1: no such row or nothing visible
  float scale;    // e^gain / sqrt(D) log2(e)
  long long row;  // token * Hq + head, -1: no such row
};

template <class E, int DT>
__device__ __forceinline__ Rows<E, DT> load_rows(const PagedAttnIO& io, const SeqSpan& sp, int h, int r) {
  typedef Tile<E, DT> P;
  Rows<E, DT> R;
  const int G4 = (threadIdx.x >> 4) & 3;
  const int D = io.c.D;
  const bool ok = r < sp.n * io.group;
  const int t = ok ? r / io.group : 0;
  const int head = h * io.group + (ok ? r - t * io.group : 0);
  R.pos = ok ? sp.len - sp.n + t : -1;
  R.scale = head_scale_log2(io.log_gain, head, D);
  R.row = ok ? (long long)(sp.t0 + t) * io.Hq + head : -1;
  const E* q = static_cast<const E*>(io.q) + (long long)(sp.t0 + t) * io.q_ts + (long long)head * io.q_hs;
#pragma unroll
  for (int p = 0; p < P::kPieces; ++p) {
    const int d = DT / 4 * G4 + P::kVec * p;
    R.q[p] = ok && d < D ? *reinterpret_cast<const u32x4*>(q + d) : u32x4{0, 0, 0, 0};
  }
  return R;
}

// K rows of a lane: slots 8 (i / 4) + 4 b + i % 4 of a tile, i = lane % 16, b = 0, 1.
template <class E, int DT> struct KRows {
  u32x4 k[2][Tile<E, DT>::kPieces];
};
__device__ __forceinline__ int k_slot(int b) {
  const int i = threadIdx.x & 15;
  return 8 * (i >> 2) + 4 * b + (i & 3);
}
// Where a slot's row lies: the page's number is loaded first, the row's data
// through it a tile later.
struct RowRef {
  int page, row;
};
// A page number as it is followed: one outside the cache (bad_pages) as page 0.
__device__ __forceinline__ int page_in(const PagedCache& c, int page) {
  return (unsigned)page < (unsigned)c.num_pages ? page : 0;
}
__device__ __forceinline__ RowRef row_ref(const PagedCache& c, const int* table, int key, int last) {
  key = key < 0 ? 0 : key > last ? last : key;
  const int idx = page_of(c.div, key);
  return RowRef{page_in(c, table[idx]), key - idx * (int)c.div.size};
}
__device__ __forceinline__ long long row_at(const PagedCache& c, RowRef r) {
  return (long long)r.page * c.page_stride + (long long)r.row * c.row_stride;
}
template <class E, int DT>
__device__ __forceinline__ void load_k(const PagedCache& c, const E* kh, const RowRef (&ref)[2],
                                       KRows<E, DT>& out) {
  typedef Tile<E, DT> P;
  const int G4 = (threadIdx.x >> 4) & 3;
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const E* p = kh + row_at(c, ref[b]);
#pragma unroll
    for (int j = 0; j < P::kPieces; ++j) {
      const int d = DT / 4 * G4 + P::kVec * j;
      out.k[b][j] = d < c.D ? *reinterpret_cast<const u32x4*>(p + d) : u32x4{0, 0, 0, 0};
    }
  }
}
// Scores q . k of the lane's query and its eight slots, unscaled.
template <class E, int DT>
__device__ __forceinline__ void add_products(const KRows<E, DT>& kr, const Rows<E, DT>& R, f32x4 (&acc)[2]) {
  typedef Tile<E, DT> P;
#pragma unroll
  for (int p = 0; p < P::kPieces; ++p) {
    if constexpr (P::kF32) {
      const f32x4 q = __builtin_bit_cast(f32x4, R.q[p]);
      const f32x4 k0 = __builtin_bit_cast(f32x4, kr.k[0][p]), k1 = __builtin_bit_cast(f32x4, kr.k[1][p]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        acc[0] = mfma16_f32(k0[e], q[e], acc[0]);
        acc[1] = mfma16_f32(k1[e], q[e], acc[1]);
      }
    } else {
      acc[0] = mfma16_of(kr.k[0][p], R.q[p], acc[0], (const E*)nullptr);
      acc[1] = mfma16_of(kr.k[1][p], R.q[p], acc[1], (const E*)nullptr);
    }
  }
}
template <class E, int DT>
__device__ __forceinline__ void tile_products(const KRows<E, DT>& kr, const Rows<E, DT>& R, float (&s)[8]) {
  f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
  add_products<E, DT>(kr, R, acc);
#pragma unroll
  for (int r = 0; r < 8; ++r) s[r] = acc[r >> 2][r & 3];
}

// Weights of the lane's eight slots of a tile that owns the 30 in its middle (slots
// 0 and 31 are the neighbours whose segments reach into it, so that no tile
// depends on another; 6.7% is done twice) from their scores relative to the row's
// shift (log2 units, the factor 4 of the segment math taken off as there, so
// that weights are in units of 2^shift).  key0: key of the lane's first slot.
// MASK: some slot of the tile is before key 0 or behind a row's own key.
template <bool MASK>
__device__ __forceinline__ void tile_weights(const float (&s)[8], int key0, int pos, float (&w)[8]) {
  const int G4 = (threadIdx.x >> 4) & 3;
  float sl = row_before(s[7]);
  float pl = fast_exp2(sl);
  float l0 = 0.f;
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const float sr = s[r];
    const float pr = fast_exp2(sr);
    float L, R;
    seg_shares(sl, sr, pl, pr, L, R);
    const int key = key0 + r;
    bool ok = r > 0 || G4 > 0;  // slot 0 has no left neighbour in the tile
    if (MASK) ok = ok && key >= 1 && key <= pos;
    if (MASK || r == 0) {
      L = ok ? L : 0.f;
      R = ok ? R : 0.f;
    }
    if (r == 0) l0 = L; else w[r - 1] += L;
    w[r] = R;
    if (MASK) {
      const float cap = 2.0f * pr;
      w[r] += key == 0 && pos >= 0 ? cap : 0.f;
      w[r] += key == pos && pos >= 0 ? cap : 0.f;
    }
    sl = sr;
    pl = pr;
  }
  const float lb = row_behind(l0);
  w[7] += lb;
  // the neighbours are another tile's
  w[0] = G4 == 0 ? 0.f : w[0];
  w[7] = G4 == 3 ? 0.f : w[7];
}

// The same where the lane's eight keys have neighbours on both sides (sl, sr,
// relative like s): every key is the lane's own.
template <bool MASK>
__device__ __forceinline__ void span_weights(const float (&s)[8], float sl, float s_end, int key0, int pos,
                                             float (&w)[8]) {
  float pl = fast_exp2(sl);
#pragma unroll
  for (int r = 0; r < 9; ++r) {
    const float sr = r < 8 ? s[r] : s_end;
    const float pr = fast_exp2(sr);
    float L, R;
    seg_shares(sl, sr, pl, pr, L, R);
    const int key = key0 + r;
    if (MASK) {
      const bool ok = key >= 1 && key <= pos;
      L = ok ? L : 0.f;
      R = ok ? R : 0.f;
    }
    if (r > 0) w[r - 1] += L;
    if (r < 8) {
      w[r] = R;
      if (MASK) {
        const float cap = 2.0f * pr;
        w[r] += key == 0 && pos >= 0 ? cap : 0.f;
        w[r] += key == pos && pos >= 0 ? cap : 0.f;
      }
    }
    sl = sr;
    pl = pr;
  }
}

// The weights of the eight keys before the lane's scores' (key skey - 1 + r in
// w[r], skey the key of s[0]) but for the right share that w[0] gets from its own
// segment; returns the one that the key of s[7] gets.  sl: the score of w[0]'s key.
template <bool MASK>
__device__ __forceinline__ float shared_weights(const float (&s)[8], float sl, int skey, int pos, float (&w)[8]) {
  float pl = fast_exp2(sl), from_left = 0.f;
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const float sr = s[r];
    const float pr = fast_exp2(sr);
    float L, R;
    seg_shares(sl, sr, pl, pr, L, R);
    const int key = skey + r;
    if (MASK) {
      const bool ok = key <= pos;
      L = ok ? L : 0.f;
      R = ok ? R : 0.f;
    }
    w[r] = L + from_left;
    if (MASK) {
      const float cap = 2.0f * pl;
      w[r] += key == 1 && pos >= 0 ? cap : 0.f;
      w[r] += key - 1 == pos && pos >= 0 ? cap : 0.f;
    }
    from_left = R;
    sl = sr;
    pl = pr;
  }
  return from_left;
}

// One wave's running softmax: shift (log2 units, whole), sum of weights (this
// lane's part) and O^T, whose lane holds columns 16 b + 4 G4 + e of its query.
template <int DT> struct Running {
  float m, z;
  f32x4 o[DT / 16];
};

// Anything not finite among the 16 bytes?
__device__ __forceinline__ bool any_special(u32x4 x, const float*) {
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) bad = bad || (x[e] & 0x7f800000u) == 0x7f800000u;
  return bad;
}
template <class E>
__device__ __forceinline__ bool any_special(u32x4 x, const E*) {
  constexpr unsigned kExp = std::is_same<E, __bf16>::value ? 0x7f80u : 0x7c00u;
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    bad = bad || (x[e] & kExp) == kExp || ((x[e] >> 16) & kExp) == kExp;
  return bad;
}

// The finite ones of packed 16-bit values, 0 for the others.
template <class E>
__device__ __forceinline__ u32x4 finite_part(u32x4 x) {
  constexpr unsigned kExp = std::is_same<E, __bf16>::value ? 0x7f80u : 0x7c00u;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if ((x[e] & kExp) == kExp) x[e] &= 0xffff0000u;
    if ((x[e] >> 16 & kExp) == kExp) x[e] &= 0xffffu;
  }
  return x;
}
__device__ __forceinline__ bool is_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// Weights in two 16-bit limbs, as an operand.
template <class E> struct Limbs16 {
  u32x4 hi, lo;
};
template <class E>
__device__ __forceinline__ Limbs16<E> limbs16(const float (&w)[8]) {
  Limbs16<E> r;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const float a = w[2 * p], b = w[2 * p + 1];
    if constexpr (std::is_same<E, __bf16>::value) {
      unsigned x[3];
      split_pair_limbs<2>(a, b, x);
      r.hi[p] = x[0];
      r.lo[p] = x[1];
    } else {
      typedef __fp16 h2 __attribute__((ext_vector_type(2)));
      const h2 h = __builtin_amdgcn_cvt_pkrtz(a, b);
      const h2 l = __builtin_amdgcn_cvt_pkrtz(a - (float)h[0], b - (float)h[1]);
      r.hi[p] = __builtin_bit_cast(unsigned, h);
      r.lo[p] = __builtin_bit_cast(unsigned, l);
    }
  }
  return r;
}

// O^T += V^T W^T over the tile's 32 slots; vs: the tile's V rows; the weights as
// they are (fp32) or in limbs.  FINITE: without the values that are not finite.
template <class E, int DT, bool FINITE>
__device__ __forceinline__ void add_values(Running<DT>& st, const E* vs, const float (&w)[8],
                                           const Limbs16<E>& wl) {
  typedef Tile<E, DT> P;
  const int lane = threadIdx.x & 63, i = lane & 15, G4 = lane >> 4;
  if constexpr (P::kF32) {
#pragma unroll
    for (int b = 0; b < DT / 16; ++b) {
      // formed from zero and added once: the sum's rounding does not grow
      // with the instructions of a tile
      f32x4 part = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        float v = vs[(8 * G4 + r) * P::kRow + 16 * b + i];
        if (FINITE) v = is_finite(v) ? v : 0.f;
        part = mfma16_f32(v, w[r], part);
      }
      st.o[b] += part;
    }
  } else {
    // transposed reads: see lds_read_tr8
    const __bf16* base = reinterpret_cast<const __bf16*>(vs) + (8 * G4 + (i >> 2)) * P::kRow + 4 * (i & 3);
#pragma unroll
    for (int b = 0; b < DT / 16; ++b) {
      u32x4 a = __builtin_bit_cast(u32x4, lds_read_tr8(base + 16 * b, base + 4 * P::kRow + 16 * b));
      if (FINITE) a = finite_part<E>(a);
      st.o[b] = mfma16_of(a, wl.lo, st.o[b], (const E*)nullptr);
      st.o[b] = mfma16_of(a, wl.hi, st.o[b], (const E*)nullptr);
    }
  }
}
// The values that are not finite, key by key, into the rows that see them: in a
// tile that some row sees only in part, a product with their zero weights would
// carry them into rows that must not read them.  Those rows' sums stay as they
// would be with any other values there, bit for bit.
template <class E, int DT>
__device__ __forceinline__ void add_values_seen(Running<DT>& st, const E* vs, const float (&w)[8], int tile_key,
                                                int pos, int first_slot, int end_slot) {
  typedef Tile<E, DT> P;
  const int lane = threadIdx.x & 63, i = lane & 15, G4 = lane >> 4;
#pragma unroll
  for (int r = 0; r < 8; ++r)
    for (int g = 0; g < 4; ++g) {
      const int slot = 8 * g + r;
      const float x = __shfl(w[r], 16 * g + i);
      const bool seen = slot >= first_slot && slot < end_slot && tile_key + slot <= pos;
#pragma unroll
      for (int b = 0; b < DT / 16; ++b) {
        const f32x4 v = ld4(vs + slot * P::kRow + 16 * b + 4 * G4);
#pragma unroll
        for (int e = 0; e < 4; ++e) st.o[b][e] += seen && !is_finite(v[e]) ? x * v[e] : 0.f;
      }
    }
}

// The same in fp32 with V from memory (shared memory holds limbs of the finite ones).
template <int DT>
__device__ __forceinline__ void add_specials(Running<DT>& st, const float* vh, const PagedCache& c,
                                             const int* table, const float (&w)[8], int k0, int end, int pos,
                                             int pos_max) {
  const int lane = threadIdx.x & 63, i = lane & 15, G4 = lane >> 4;
#pragma unroll
  for (int r = 0; r < 8; ++r)
    for (int g = 0; g < 4; ++g) {
      const int key = k0 + 8 * g + r;
      const float x = __shfl(w[r], 16 * g + i);
      if (key >= end) continue;  // uniform
      const float* v = vh + row_at(c, row_ref(c, table, key, pos_max));
#pragma unroll
      for (int b = 0; b < DT / 16; ++b) {
        if (16 * b + 4 * G4 >= c.D) continue;
        const f32x4 y = ld4(v + 16 * b + 4 * G4);
#pragma unroll
        for (int e = 0; e < 4; ++e) st.o[b][e] += key <= pos && !is_finite(y[e]) ? x * y[e] : 0.f;
      }
    }
}

__device__ __forceinline__ float nan_value() { return __int_as_float(0x7fc00000); }

// Does this thread's share of the page numbers of slots [first, last] hold one
// outside the cache?  What reads through it is NaN in the end; loads meanwhile
// follow page_in and need not wait for the answer.
__device__ __forceinline__ bool bad_pages(const PagedCache& c, const int* table, int first, int last) {
  bool bad = false;
  const int end = page_of(c.div, last);
  for (int i = page_of(c.div, first) + (int)threadIdx.x; i <= end; i += (int)blockDim.x)
    bad = bad || (unsigned)table[i] >= (unsigned)c.num_pages;
  return bad;
}

// Many rows: WV waves of 16 rows each share the tiles of V.  A weight tile is the
// 32 keys from k0 on, its score tile the 32 from k0 + 1 on (slot x of the scores
// is key k0 + 1 + x): the segment that ends at a score's key gives its left share
// to the weight in the same register and its right share to the next one, the
// last one of a tile to the next tile, as in the training forward.  So nothing is
// done twice but for the segment that crosses a split's start, which comes from
// one product of its own.  Tiles start at multiples of 32, as for few rows.
//
// fp32 goes through three bf16 limbs here: K and V are split once for all of the
// waves when they are staged, and six bf16 products take 40% of the time of one
// on the fp32 instruction (two prompts of 2048 tokens 310 -> 202 us).  (Few rows
// keep the fp32 instruction: there each wave would split what it reads.)  Not
// kept: 16 waves a work group (197 against 196 us) and K's limbs in the order the
// instruction reads them (half the bank conflicts, no time).
template <class E, int DT, int WV> struct Many {
  typedef Tile<E, DT> P;
  static constexpr int kThreads = 64 * WV, kRows = 16 * WV;
  static constexpr int kChunks = 32 * P::kChunks;                       // 16-byte chunks of a tile
  static constexpr int kLoads = (kChunks + kThreads - 1) / kThreads;   // of each thread
  static constexpr int kLRow = DT + 16;                                 // staged row of bf16
  static constexpr int kPlane = 32 * kLRow;
  // V of two tiles; fp32: limb planes of K and V of two tiles
  static constexpr int kBytes = 2 * (P::kF32 ? 6 * kPlane * 2 : 32 * P::kRow * 2);
};

// Waves per SIMD that the registers are held to.  Four at up to 64 columns, though
// that spills a few (16-bit 4 to 24, fp32 27 at most): with three, one work group of
// eight waves is left per CU (512 tokens over 8192 in bf16 116 -> 175 us, two fp32
// prompts of 2048 tokens 208 -> 232).
template <int DT> constexpr int many_waves() { return DT <= 64 ? 4 : 2; }

template <class E, int DT, int WV, bool PAGE32>
__global__ __launch_bounds__(64 * WV, (many_waves<DT>())) void ca_paged_attention_kernel(PagedAttnIO io) {
  typedef Tile<E, DT> P;
  typedef Many<E, DT, WV> M;
  constexpr int KS = DT / 32;  // 32-wide products of the scores in limbs
  __shared__ __attribute__((aligned(16))) unsigned char lds[M::kBytes];
  __shared__ int special[2];  // tile (plus one) whose V holds a value that is not finite

  const PagedCache& c = io.c;
  const int tid = threadIdx.x, lane = tid & 63, i16 = lane & 15, G4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int slices = c.batch * c.heads;
  // slices fastest: a slice's work groups meet on one XCD when slices are a
  // multiple of eight
  const int slice = blockIdx.x % slices, rest = blockIdx.x / slices;
  const int split = rest % io.splits, tile0 = rest / io.splits;
  const int b = slice / c.heads, h = slice - b * c.heads;
  const SeqSpan sp = seq_span(c, b, io.tokens);
  const int rows = sp.n * io.group;
  const int* table = c.table + (long long)b * c.table_stride;
  const E* kh = static_cast<const E*>(c.k) + (long long)h * c.head_stride;
  const E* vh = static_cast<const E*>(c.v) + (long long)h * c.head_stride;
  const int row_tiles = (rows + M::kRows - 1) / M::kRows;
  const int rs = (int)c.row_stride;  // (PAGE32: below 2^25)

  // longest rows first
  for (int back = tile0; back < row_tiles; back += io.row_tiles) {
    const int row0 = (row_tiles - 1 - back) * M::kRows;
    const int last_row = row0 + M::kRows < rows ? row0 + M::kRows - 1 : rows - 1;
    const int pos_max = sp.len - sp.n + last_row / io.group;  // last slot any row sees
    const int pos_min = sp.len - sp.n + row0 / io.group;
    const int first = split * io.split_keys;
    if (pos_max < first && split > 0) continue;  // nothing here; the join knows
    const int end = split == io.splits - 1 || first + io.split_keys > pos_max ? pos_max + 1 : first + io.split_keys;
    const int ntiles = end > first ? (end - first + 31) / 32 : 0;
    const bool whole_rows = io.splits == 1 || pos_max < io.split_keys;  // this split is all they see
    // (fp32: the quarter rows feed the product at the split's start, the limbs the tiles)
    const Rows<E, DT> R = load_rows<E, DT>(io, sp, h, row0 + 16 * wave + i16);
    Limbs qb[P::kF32 ? KS : 1];
    if constexpr (P::kF32) {
      const float* q = static_cast<const float*>(io.q);
      if (R.row >= 0) q += (R.row / io.Hq) * io.q_ts + (R.row % io.Hq) * io.q_hs;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          const int d = 32 * ks + 8 * G4 + e;
          const f32x4 v = R.row >= 0 && d < c.D ? ld4(q + d) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int f = 0; f < 4; ++f) x[e + f] = v[f];
        }
        qb[ks] = split8(x);
      }
    }
    Running<DT> st;
    st.m = kNegBig;
    st.z = 0.f;
#pragma unroll
    for (int x = 0; x < DT / 16; ++x) st.o[x] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (tid < 2) special[tid] = 0;
    bool bad = false;
    if (ntiles > 0) {
      bad = bad_pages(c, table, first > 0 ? first - 1 : 0, end <= pos_max ? end : pos_max);
      // ---- where rows lie ----
      auto clamped = [&](int key) { return key < 0 ? 0 : key > pos_max ? pos_max : key; };
      auto page_at = [&](int key) { return page_in(c, table[page_of(c.div, clamped(key))]); };
      // of a key whose page's number is known
      auto in_page = [&](int key, int page) {
        const int at = clamped(key), idx = page_of(c.div, at);
        return (long long)__builtin_amdgcn_readfirstlane(page) * c.page_stride +
               (long long)(at - idx * (int)c.div.size) * c.row_stride;
      };
      int page0 = 0, page1 = 0;  // PAGE32: of the tile to be loaded next, and of the one behind it
      RowRef kref[P::kF32 ? M::kLoads : 2], vref[M::kLoads];
      auto look_up = [&](int k0) {  // of the tile to be loaded next
        if constexpr (PAGE32) {
          page0 = page1;
          page1 = page_at(k0 + 32);
        } else {
#pragma unroll
          for (int x = 0; x < (P::kF32 ? M::kLoads : 2); ++x)
            kref[x] = row_ref(c, table, k0 + 1 + (P::kF32 ? (tid + x * M::kThreads) / P::kChunks : k_slot(x)), pos_max);
#pragma unroll
          for (int x = 0; x < M::kLoads; ++x)
            vref[x] = row_ref(c, table, k0 + (tid + x * M::kThreads) / P::kChunks, pos_max);
        }
      };
      // ---- loads of a tile ----
      KRows<E, DT> kr;                // 16-bit: the wave's operand
      u32x4 kreg[M::kLoads], vreg[M::kLoads];  // what this thread stages (kreg: fp32)
      auto load_tile = [&](int k0) {
        long long at0 = 0, at1 = 0;
        if constexpr (PAGE32) {
          at0 = in_page(k0, page0);
          at1 = in_page(k0 + 32, page1);
        }
        if constexpr (!P::kF32) {
          const int d0 = DT / 4 * G4;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const E* p;
            if constexpr (PAGE32)
              p = kh + (k_slot(x) == 31 ? at1 + d0 : at0 + ((k_slot(x) + 1) * rs + d0));
            else
              p = kh + row_at(c, kref[x]) + d0;
#pragma unroll
            for (int j = 0; j < P::kPieces; ++j)
              kr.k[x][j] = d0 + P::kVec * j < c.D ? *reinterpret_cast<const u32x4*>(p + P::kVec * j) : u32x4{0, 0, 0, 0};
          }
        }
        const bool whole = k0 + 32 <= end;
#pragma unroll
        for (int x = 0; x < M::kLoads; ++x) {
          const int u = tid + x * M::kThreads, row = u / P::kChunks, d = u % P::kChunks * P::kVec;
          // V: keys behind the last one stay out: zeros
          const bool mine = row < 32 && d < c.D && (whole || k0 + row < end);
          const E* p;
          if constexpr (PAGE32) p = vh + at0 + (row * rs + d);
          else p = vh + row_at(c, vref[x]) + d;
          vreg[x] = mine ? *reinterpret_cast<const u32x4*>(p) : u32x4{0, 0, 0, 0};
          if constexpr (P::kF32) {
            if constexpr (PAGE32) p = kh + (row == 31 ? at1 + d : at0 + ((row + 1) * rs + d));
            else p = kh + row_at(c, kref[x]) + d;
            kreg[x] = row < 32 && d < c.D ? *reinterpret_cast<const u32x4*>(p) : u32x4{0, 0, 0, 0};
          }
        }
      };
      auto stage = [&](int t, int buf) {
        const bool look = first + 32 * (t + 1) > pos_min;
#pragma unroll
        for (int x = 0; x < M::kLoads; ++x) {
          const int u = tid + x * M::kThreads, row = u / P::kChunks, d = u % P::kChunks * P::kVec;
          if (M::kChunks % M::kThreads != 0 && row >= 32) continue;
          if constexpr (P::kF32) {
            __bf16* kp = reinterpret_cast<__bf16*>(lds) + buf * 6 * M::kPlane;
            const f32x4 kv = __builtin_bit_cast(f32x4, kreg[x]);
            f32x4 vv = __builtin_bit_cast(f32x4, vreg[x]);
            bool odd = false;
            if (look) {
              // values that are not finite stay out of the limbs, for the rows
              // that see them to add by themselves
#pragma unroll
              for (int e = 0; e < 4; ++e) odd = odd || !is_finite(vv[e]);
              if (odd) special[buf] = t + 1;
#pragma unroll
              for (int e = 0; e < 4; ++e) vv[e] = is_finite(vv[e]) ? vv[e] : 0.f;
            }
            unsigned k0w[3], k1w[3], v0w[3], v1w[3];
            split_pair_limbs<3>(kv[0], kv[1], k0w);
            split_pair_limbs<3>(kv[2], kv[3], k1w);
            split_pair_limbs<3>(vv[0], vv[1], v0w);
            split_pair_limbs<3>(vv[2], vv[3], v1w);
#pragma unroll
            for (int l = 0; l < 3; ++l) {
              *reinterpret_cast<u32x2*>(kp + l * M::kPlane + row * M::kLRow + d) = u32x2{k0w[l], k1w[l]};
              *reinterpret_cast<u32x2*>(kp + (3 + l) * M::kPlane + row * M::kLRow + d) = u32x2{v0w[l], v1w[l]};
            }
          } else {
            *reinterpret_cast<u32x4*>(reinterpret_cast<E*>(lds) + (buf * 32 + row) * P::kRow + d) = vreg[x];
            if (look && any_special(vreg[x], (const E*)nullptr)) special[buf] = t + 1;
          }
        }
      };

      // ---- the split's start: the scores of its first key and of the one before ----
      // Scores are kept relative to shift = m + kAbove (see tile_weights).
      constexpr float kAbove = kShareShift - weight_octaves<E>();
      float shift, s_carry, r_carry = 0.f;  // score of the tile's first key, right share it gets
      {
        const int key = (i16 & 3) == 1 ? first - 1 : first;
        const RowRef ref = row_ref(c, table, key, pos_max);
        const E* p = kh + row_at(c, ref) + DT / 4 * G4;
        f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
        if constexpr (PAGE32) page1 = page_at(first);
        look_up(first);
        load_tile(first);
#pragma unroll
        for (int j = 0; j < P::kPieces; ++j) {
          const bool in = DT / 4 * G4 + P::kVec * j < c.D;
          const u32x4 k = in ? *reinterpret_cast<const u32x4*>(p + P::kVec * j) : u32x4{0, 0, 0, 0};
          if constexpr (P::kF32) {
            const f32x4 a = __builtin_bit_cast(f32x4, k), q = __builtin_bit_cast(f32x4, R.q[j]);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc = mfma16_f32(a[e], q[e], acc);
          } else {
            acc = mfma16_of(k, R.q[j], acc, (const E*)nullptr);
          }
        }
        const float at = acc[0] * R.scale, before = acc[1] * R.scale;
        const bool sees = first <= R.pos, seg = sees && first > 0;
        // (rows that see nothing yet never will in this split; from a score that
        // is not finite no shift can start)
        const float top = seg ? fmaxf(at, before) : at;
        shift = (sees && is_finite(top) ? rintf(top) : 0.f) + kAbove;
        s_carry = at - shift;
        const float sl = before - shift;
        float L, Rs;
        seg_shares(sl, s_carry, fast_exp2(sl), fast_exp2(s_carry), L, Rs);
        r_carry = seg ? Rs : 0.f;
        __syncthreads();  // `special` has been cleared
        stage(0, 0);
        if (ntiles > 1) look_up(first + 32);
      }
      __syncthreads();

      for (int t = 0; t < ntiles; ++t) {
        const int buf = t & 1, k0 = first + 32 * t;
        float s[8], w[8];
        if constexpr (P::kF32) {
          const __bf16* kp = reinterpret_cast<const __bf16*>(lds) + buf * 6 * M::kPlane;
          f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            Limbs ka[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) ka[x] = limbs_at<3>(kp + k_slot(x) * M::kLRow + 32 * ks + 8 * G4, M::kPlane);
#pragma unroll
            for (int step = 0; step < 6; ++step) {
              acc[0] = mfma16_step(step, ka[0], qb[ks], acc[0]);
              acc[1] = mfma16_step(step, ka[1], qb[ks], acc[1]);
            }
          }
#pragma unroll
          for (int r = 0; r < 8; ++r) s[r] = acc[r >> 2][r & 3];
        } else {
          tile_products<E, DT>(kr, R, s);
        }
        if (t + 1 < ntiles) {
          load_tile(k0 + 32);
          if (t + 2 < ntiles) look_up(k0 + 64);
        }
        const int skey = k0 + 1 + 8 * G4;  // key of s[0]; w[0]'s is the one before
        const bool mask = k0 == 0 || k0 + 32 > pos_min;
        // relative to the shift so far, which a tile seldom moves
        float mt = kNegBig;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          s[r] = fmaf(s[r], R.scale, -shift);
          mt = fmaxf(mt, !mask || skey + r <= R.pos ? s[r] : kNegBig);
        }
        mt = rows_max(mt);
        const bool grow = mt > kLazyRescale - kAbove;
        if (wave_any(grow)) {
          const float up = grow ? rintf(mt + kAbove) : 0.f;
          const float alpha = fast_exp2(-up);
#pragma unroll
          for (int x = 0; x < DT / 16; ++x) st.o[x] *= alpha;
          st.z *= alpha;
          r_carry *= alpha;
          s_carry -= up;
          shift += up;
#pragma unroll
          for (int r = 0; r < 8; ++r) s[r] -= up;
        }
        const float s_last = row_before(s[7]);  // lane row 0: the next tile's carry
        const float sl0 = G4 == 0 ? s_carry : s_last;
        s_carry = s_last;
        float r_out = mask ? shared_weights<true>(s, sl0, skey, R.pos, w) : shared_weights<false>(s, sl0, skey, R.pos, w);
        r_out = row_before(r_out);
        w[0] += G4 == 0 ? r_carry : r_out;
        r_carry = r_out;
#pragma unroll
        for (int r = 0; r < 8; ++r) st.z += w[r];
        if constexpr (P::kF32) {
          const __bf16* vp = reinterpret_cast<const __bf16*>(lds) + (buf * 6 + 3) * M::kPlane;
          const __bf16* base = vp + (8 * G4 + (i16 >> 2)) * M::kLRow + 4 * (i16 & 3);
          const Limbs wb = split8(w);
#pragma unroll
          for (int x = 0; x < DT / 16; x += 2) {
            f32x4 part[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
            Limbs va[2];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const __bf16* at = base + 16 * (x + y);
              va[y].h = lds_read_tr8(at, at + 4 * M::kLRow);
              va[y].m = lds_read_tr8(at + M::kPlane, at + M::kPlane + 4 * M::kLRow);
              va[y].l = lds_read_tr8(at + 2 * M::kPlane, at + 2 * M::kPlane + 4 * M::kLRow);
            }
#pragma unroll
            for (int step = 0; step < 6; ++step) {
              part[0] = mfma16_step(step, va[0], wb, part[0]);
              part[1] = mfma16_step(step, va[1], wb, part[1]);
            }
            // a tile's product is added once: its rounding does not grow with the sum
            st.o[x] += part[0];
            st.o[x + 1] += part[1];
          }
          if (mask && special[buf] == t + 1) add_specials<DT>(st, vh, c, table, w, k0, end, R.pos, pos_max);
        } else {
          const Limbs16<E> wl = limbs16<E>(w);
          const E* vs = reinterpret_cast<const E*>(lds) + buf * 32 * P::kRow;
          if (mask && special[buf] == t + 1) {
            add_values<E, DT, true>(st, vs, w, wl);
            add_values_seen<E, DT>(st, vs, w, k0, R.pos, 0, 32);
          } else {
            add_values<E, DT, false>(st, vs, w, wl);
          }
        }
        if (t + 1 < ntiles) stage(t + 1, buf ^ 1);
        __syncthreads();
      }
      st.z = rows_sum(st.z);
      st.m = first <= R.pos ? shift - kAbove : kNegBig;
    }
    if (__syncthreads_or(bad)) st.m = st.z = nan_value();

    const long long nrows = (long long)io.tokens * io.Hq;
    const float meff = st.m - weight_octaves<E>();
    if (R.row >= 0) {
      if (whole_rows) {
        const float inv = st.z == 0.f ? 0.f : 1.0f / st.z;
        E* o = static_cast<E*>(io.out) + (R.row / io.Hq) * io.o_ts + (R.row % io.Hq) * io.o_hs;
#pragma unroll
        for (int x = 0; x < DT / 16; ++x)
          if (16 * x + 4 * G4 < c.D) st4(o + 16 * x + 4 * G4, st.o[x] * inv);
        if (io.stats && G4 == 0) {
          io.stats[2 * R.row] = meff;
          io.stats[2 * R.row + 1] = inv;
        }
      } else {
        float* o = io.part_o + (split * nrows + R.row) * c.D;
#pragma unroll
        for (int x = 0; x < DT / 16; ++x)
          if (16 * x + 4 * G4 < c.D) st4(o + 16 * x + 4 * G4, st.o[x]);
        if (G4 == 0) {
          io.part_ml[2 * (split * nrows + R.row)] = meff;
          io.part_ml[2 * (split * nrows + R.row) + 1] = st.z;
        }
      }
    }
    __syncthreads();  // the next row tile stages over this one's
  }
}

// Few rows: up to 8 per key head (fp32: 16).  One token of one head would leave 15 of a
// tile's 16 columns empty, and the segment math is the longest part of a tile, so
// the columns hold RP = 2^row_log rows times TP tiles of 32 keys: column c is row
// c % RP over tile c / RP of a group of TP tiles.  The group's scores come from TP
// products, of each of which the columns of its tile are kept (added up with the
// other columns' queries zeroed, a key that is not finite, behind the last one say,
// would make other keys' scores NaN); the segments are then formed once for all of the group; and O^T
// takes TP products again, each with the weights of its own columns.  Every
// column keeps its own running maximum, and columns and waves are joined at the
// end.  Per tile this leaves some 60 vector instructions of 520 with one tile at
// a time, so that the bytes bound it.
//
// Tiles here own all of their 32 keys: neighbours are other columns' scores, and
// the two beyond the group come from one more product (K rows k0 - 1 and k0 + 32 TP).
// So tiles start at multiples of 32, and where pages hold a multiple of 16 slots
// (PAGE16) half a tile lies in one page: its number is read once for the wave and
// addresses are a scalar base and a constant offset per lane.
template <class E, int DT> struct Few {
  typedef Tile<E, DT> P;
  static constexpr int kV = 32 * P::kChunks / 64;  // 16-byte pieces of V of a lane per tile
};
template <class E, int DT> struct VRows {
  u32x4 v[Few<E, DT>::kV];
};

template <class E, int DT, bool PAGE16>
__global__ __launch_bounds__(256) void ca_paged_few_kernel(PagedAttnIO io) {
  typedef Tile<E, DT> P;
  constexpr int kV = Few<E, DT>::kV;
  constexpr int kVBytes = 4 * 32 * P::kRow * (int)sizeof(E);
  constexpr int kJRow = DT + 4;
  constexpr int kJoinBytes = 4 * 16 * kJRow * (int)sizeof(float);
  __shared__ __attribute__((aligned(16))) unsigned char lds[kVBytes > kJoinBytes ? kVBytes : kJoinBytes];

  const PagedCache& c = io.c;
  const int tid = threadIdx.x, lane = tid & 63, i16 = lane & 15, G4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int slices = c.batch * c.heads;
  const int slice = blockIdx.x % slices, rest = blockIdx.x / slices;
  const int split = rest % io.splits, tile0 = rest / io.splits;
  const int b = slice / c.heads, h = slice - b * c.heads;
  const SeqSpan sp = seq_span(c, b, io.tokens);
  const int rows = sp.n * io.group;
  const int* table = c.table + (long long)b * c.table_stride;
  const E* kh = static_cast<const E*>(c.k) + (long long)h * c.head_stride;
  const E* vh = static_cast<const E*>(c.v) + (long long)h * c.head_stride;
  const int RP = 1 << io.row_log, TP = io.tile_group;
  const int row_tiles = (rows + RP - 1) >> io.row_log;
  const int u_col = i16 >> io.row_log;  // the tile of this lane's column
  const int k_d = DT / 4 * G4;          // first of the lane's D values of K
  E* vs = reinterpret_cast<E*>(lds) + wave * 32 * P::kRow;

  for (int back = tile0; back < row_tiles; back += io.row_tiles) {
    const int row0 = (row_tiles - 1 - back) << io.row_log;
    const int last_row = row0 + RP < rows ? row0 + RP - 1 : rows - 1;
    const int pos_max = sp.len - sp.n + last_row / io.group;
    const int pos_min = sp.len - sp.n + row0 / io.group;
    const int first = split * io.split_keys;
    if (pos_max < first && split > 0) continue;  // the join knows
    const int end = split == io.splits - 1 || first + io.split_keys > pos_max ? pos_max + 1 : first + io.split_keys;
    const bool whole_rows = io.splits == 1 || pos_max < io.split_keys;  // this split is all they see
    const Rows<E, DT> R = load_rows<E, DT>(io, sp, h, row0 + (i16 & (RP - 1)));
    Running<DT> st;
    st.m = kNegBig;
    st.z = 0.f;
#pragma unroll
    for (int x = 0; x < DT / 16; ++x) st.o[x] = f32x4{0.f, 0.f, 0.f, 0.f};
    bool bad = false;
    if (end > first) {
      bad = bad_pages(c, table, first > 0 ? first - 1 : 0, end <= pos_max ? end : pos_max);
      const int step = 32 * TP;
      // Page numbers of a group: lane x < 32 those of its halves of tiles, lanes 32
      // and 33 the neighbours'.  (Only what PAGE16 needs.)
      auto group_pages = [&](int k0) {
        int key = lane < 32 ? k0 + 16 * lane : lane == 32 ? k0 - 1 : k0 + step;
        key = key < 0 ? 0 : key > pos_max ? pos_max : key;
        return page_in(c, table[page_of(c.div, key)]);
      };
      int ids = 0, next_ids = 0;
      auto half_at = [&](int key, int x) {  // of half x of the group, its first key `key`
        const int idx = page_of(c.div, key);
        const int page = __builtin_amdgcn_readlane(ids, x);
        return (long long)page * c.page_stride + (long long)(key - idx * (int)c.div.size) * c.row_stride;
      };
      // row x of tile u lies at from[x / 16] + x row strides; rows of a half that
      // nothing sees stand for the first one's
      auto halves = [&](int key, int u, long long& from0, long long& from1) {
        from0 = half_at(key, 2 * u);
        from1 = (key + 16 <= pos_max ? half_at(key + 16, 2 * u + 1) : from0) - 16 * c.row_stride;
      };
      auto load_ktile = [&](int key, int u, KRows<E, DT>& out) {
        if constexpr (PAGE16) {
          long long from0, from1;
          halves(key, u, from0, from1);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const E* p = kh + ((k_slot(x) < 16 ? from0 : from1) + (k_slot(x) * (int)c.row_stride + k_d));
#pragma unroll
            for (int j = 0; j < P::kPieces; ++j)
              out.k[x][j] = k_d + P::kVec * j < c.D ? *reinterpret_cast<const u32x4*>(p + P::kVec * j)
                                                    : u32x4{0, 0, 0, 0};
          }
        } else {
          RowRef ref[2];
#pragma unroll
          for (int x = 0; x < 2; ++x) ref[x] = row_ref(c, table, key + k_slot(x), pos_max);
          load_k<E, DT>(c, kh, ref, out);
        }
      };
      auto load_vtile = [&](int key, int u, VRows<E, DT>& out) {
        long long from0 = 0, from1 = 0;
        if constexpr (PAGE16) halves(key, u, from0, from1);
        const bool whole = key + 32 <= end;
#pragma unroll
        for (int x = 0; x < kV; ++x) {
          const int at = lane + 64 * x, row = at / P::kChunks, d = at % P::kChunks * P::kVec;
          const bool mine = d < c.D && (whole || key + row < end);  // behind the last key: zeros
          const E* p;
          if constexpr (PAGE16) p = vh + ((row < 16 ? from0 : from1) + (row * (int)c.row_stride + d));
          else p = vh + row_at(c, row_ref(c, table, key + row, pos_max)) + d;
          out.v[x] = mine ? *reinterpret_cast<const u32x4*>(p) : u32x4{0, 0, 0, 0};
        }
      };
      int k0 = first + wave * step;
      if (PAGE16 && k0 < end) ids = group_pages(k0);
      for (; k0 < end; k0 += 4 * step) {
        const int n = (end - k0 + 31) / 32 < TP ? (end - k0 + 31) / 32 : TP;  // tiles of this group
        if (PAGE16 && k0 + 4 * step < end) next_ids = group_pages(k0 + 4 * step);
        // scores of the group, and of its two neighbours
        KRows<E, DT> ka, kb;
        u32x4 kn[P::kPieces];
        load_ktile(k0, 0, ka);
        {
          int key = i16 == 1 ? k0 + step : k0 - 1;
          key = key < 0 ? 0 : key > pos_max ? pos_max : key;
          RowRef ref;
          if constexpr (PAGE16) {
            const int idx = page_of(c.div, key);
            const int left = __builtin_amdgcn_readlane(ids, 32), right = __builtin_amdgcn_readlane(ids, 33);
            ref = RowRef{i16 == 1 ? right : left, key - idx * (int)c.div.size};
          } else {
            ref = row_ref(c, table, key, pos_max);
          }
          const E* p = kh + row_at(c, ref) + k_d;
#pragma unroll
          for (int j = 0; j < P::kPieces; ++j)
            kn[j] = k_d + P::kVec * j < c.D ? *reinterpret_cast<const u32x4*>(p + P::kVec * j) : u32x4{0, 0, 0, 0};
        }
        VRows<E, DT> v;
        // where the registers have room, V's first tile is on its way early
        constexpr bool kEarly = DT <= 64 && !P::kF32;
        if (kEarly) load_vtile(k0, 0, v);
        f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
        auto products = [&](const KRows<E, DT>& kr, int u) {
          f32x4 part[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
          add_products<E, DT>(kr, R, part);
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[x][e] = u_col == u ? part[x][e] : acc[x][e];
        };
        for (int u = 0; u < n; u += 2) {
          if (u + 1 < n) load_ktile(k0 + 32 * (u + 1), u + 1, kb);
          products(ka, u);
          if (u + 2 < n) load_ktile(k0 + 32 * (u + 2), u + 2, ka);
          if (u + 1 < n) products(kb, u + 1);
        }
        if (!kEarly) load_vtile(k0, 0, v);
        f32x4 beyond = f32x4{0.f, 0.f, 0.f, 0.f};  // lane row 0: left, right
#pragma unroll
        for (int p = 0; p < P::kPieces; ++p) {
          if constexpr (P::kF32) {
            const f32x4 a = __builtin_bit_cast(f32x4, kn[p]), q = __builtin_bit_cast(f32x4, R.q[p]);
#pragma unroll
            for (int e = 0; e < 4; ++e) beyond = mfma16_f32(a[e], q[e], beyond);
          } else {
            beyond = mfma16_of(kn[p], R.q[p], beyond, (const E*)nullptr);
          }
        }
        float s[8], w[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) s[r] = acc[r >> 2][r & 3] * R.scale;
        const int key0 = k0 + 32 * u_col + 8 * G4;
        const bool mask = k0 == 0 || k0 + step > pos_min;
        float mt = kNegBig;
#pragma unroll
        for (int r = 0; r < 8; ++r) mt = fmaxf(mt, !mask || key0 + r <= R.pos ? s[r] : kNegBig);
        mt = rows_max(mt);
        const bool grow = mt > st.m + kLazyRescale;
        if (wave_any(grow)) {
          const float m = grow ? rintf(mt) : st.m;
          const float alpha = grow ? fast_exp2(st.m - m) : 1.0f;
#pragma unroll
          for (int x = 0; x < DT / 16; ++x) st.o[x] *= alpha;
          st.z *= alpha;
          st.m = m;
        }
        // neighbours: the lane rows before and behind; past a tile's ends the
        // next columns' and past the group's the two products'
        float s_left = s[7], s_right = s[0];
        if (TP > 1) {
          s_left = __shfl(s[7], (lane & 48) | ((i16 - RP) & 15));
          s_right = __shfl(s[0], (lane & 48) | ((i16 + RP) & 15));
        }
        s_right = u_col == TP - 1 ? beyond[1] * R.scale : s_right;
        s_left = row_before(G4 == 3 ? s_left : s[7]);
        s_left = G4 == 0 && u_col == 0 ? beyond[0] * R.scale : s_left;
        s_right = row_behind(G4 == 0 ? s_right : s[0]);
        const float shift = st.m + (kShareShift - weight_octaves<E>());
#pragma unroll
        for (int r = 0; r < 8; ++r) s[r] -= shift;
        if (mask) span_weights<true>(s, s_left - shift, s_right - shift, key0, R.pos, w);
        else span_weights<false>(s, s_left - shift, s_right - shift, key0, R.pos, w);
#pragma unroll
        for (int r = 0; r < 8; ++r) st.z += w[r];
        Limbs16<E> wl;
        if constexpr (!P::kF32) wl = limbs16<E>(w);
        for (int u = 0; u < n; ++u) {
          bool special = false;
          const bool look = k0 + 32 * (u + 1) > pos_min;
#pragma unroll
          for (int x = 0; x < kV; ++x) {
            const int at = lane + 64 * x, row = at / P::kChunks, d = at % P::kChunks * P::kVec;
            *reinterpret_cast<u32x4*>(vs + row * P::kRow + d) = v.v[x];
            if (look) special = special || any_special(v.v[x], (const E*)nullptr);
          }
          wave_lds_sync();
          if (u + 1 < n) load_vtile(k0 + 32 * (u + 1), u + 1, v);
          const bool mine = TP == 1 || u_col == u;
          float wu[8];
          Limbs16<E> lu = wl;
          if constexpr (P::kF32) {
#pragma unroll
            for (int r = 0; r < 8; ++r) wu[r] = mine ? w[r] : 0.f;
          } else if (TP > 1) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              lu.hi[e] = mine ? wl.hi[e] : 0u;
              lu.lo[e] = mine ? wl.lo[e] : 0u;
            }
          }
          if (look && wave_any(special)) {
            add_values<E, DT, true>(st, vs, wu, lu);
            add_values_seen<E, DT>(st, vs, w, k0 + 32 * u, mine ? R.pos : -1, 0, 32);
          } else {
            add_values<E, DT, false>(st, vs, wu, lu);
          }
          wave_lds_sync();
        }
        ids = next_ids;
      }
      st.z = rows_sum(st.z);
      // columns of one row
      for (int x = RP; x < RP * TP; x <<= 1) {
        const float pm = __shfl_xor(st.m, x), pz = __shfl_xor(st.z, x);
        const float m = fmaxf(st.m, pm);
        const float a = fast_exp2(st.m - m), e = fast_exp2(pm - m);
#pragma unroll
        for (int y = 0; y < DT / 16; ++y)
#pragma unroll
          for (int q = 0; q < 4; ++q) st.o[y][q] = st.o[y][q] * a + __shfl_xor(st.o[y][q], x) * e;
        st.z = st.z * a + pz * e;
        st.m = m;
      }
    }
    if (__syncthreads_or(bad)) st.m = st.z = nan_value();

    const long long nrows = (long long)io.tokens * io.Hq;
    {
      // join the four waves' parts: O, then m and z
      float* join = reinterpret_cast<float*>(lds);
      {
        float* p = join + (wave * 16 + i16) * kJRow;
#pragma unroll
        for (int x = 0; x < DT / 16; ++x) st4(p + 16 * x + 4 * G4, st.o[x]);
        if (G4 == 0) {
          p[DT] = st.m;
          p[DT + 1] = st.z;
        }
      }
      __syncthreads();
      constexpr int kQuads = DT / 4;
      for (int u = tid; u < RP * kQuads; u += 256) {
        const int r = u / kQuads, d = u % kQuads * 4;
        const int rr = row0 + r;
        if (rr >= rows || d >= c.D) continue;
        const int t = rr / io.group, head = h * io.group + rr - t * io.group;
        const long long row = (long long)(sp.t0 + t) * io.Hq + head;
        float m = kNegBig, z = 0.f;
        f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < 4; ++x) m = fmaxf(m, join[(x * 16 + r) * kJRow + DT]);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float* p = join + (x * 16 + r) * kJRow;
          const float a = fast_exp2(p[DT] - m);
          z += a * p[DT + 1];
          o += a * ld4(p + d);
        }
        const float meff = m - weight_octaves<E>();
        if (whole_rows) {
          const float inv = z == 0.f ? 0.f : 1.0f / z;
          st4(static_cast<E*>(io.out) + (long long)(sp.t0 + t) * io.o_ts + (long long)head * io.o_hs + d, o * inv);
          if (io.stats && d == 0) {
            io.stats[2 * row] = meff;
            io.stats[2 * row + 1] = inv;
          }
        } else {
          st4(io.part_o + (split * nrows + row) * c.D + d, o);
          if (d == 0) {
            io.part_ml[2 * (split * nrows + row)] = meff;
            io.part_ml[2 * (split * nrows + row) + 1] = z;
          }
        }
      }
      __syncthreads();  // the next row tile stages V over it
    }
  }
}

// Joins the splits of a row: DT / 4 lanes over its columns, SUB groups of them over
// the splits: one, those of a wave, or those of a work group (64 splits of 16
// rows took 9.6 us with one wave per row, 4.4 with four; two splits of 65536
// rows 23 with one, 8.5 with a group of 16 lanes).
template <class E, int DT, int SUB>
__global__ __launch_bounds__(256) void ca_paged_combine_kernel(PagedAttnIO io) {
  constexpr int kQuads = DT / 4, kWave = 64 / kQuads;  // groups of a wave
  constexpr int kRows = 256 / kQuads / SUB;            // rows of a work group
  __shared__ float join[SUB > kWave ? 4 : 1][DT + 4];
  const PagedCache& c = io.c;
  const int slices = c.batch * c.heads;
  const int slice = blockIdx.x % slices, part = blockIdx.x / slices;
  const int b = slice / c.heads, h = slice - b * c.heads;
  const SeqSpan sp = seq_span(c, b, io.tokens);
  const int rows = sp.n * io.group;
  const int d = threadIdx.x % kQuads * 4, lane_group = threadIdx.x / kQuads;
  const int sub = lane_group % SUB;
  const long long nrows = (long long)io.tokens * io.Hq;
  const int parts = gridDim.x / slices;
  for (int r0 = part * kRows; r0 < rows; r0 += kRows * parts) {
    const int r = r0 + lane_group / SUB;
    const bool ok = r < rows;
    const int t = ok ? r / io.group : 0, head = h * io.group + (ok ? r - t * io.group : 0);
    const long long row = (long long)(sp.t0 + t) * io.Hq + head;
    // every work group of the attention kernel wrote the rows of its tile up to
    // the last slot any of them sees: a row's splits are those up to its own
    // slot; a tile that one split covers wrote its results itself
    const int tile_end = (r / io.tile_rows + 1) * io.tile_rows;
    const int tile_last = (tile_end < rows ? tile_end : rows) - 1;
    const bool done = !ok || sp.len - sp.n + tile_last / io.group < io.split_keys;
    const int pos = sp.len - sp.n + t;
    int ns = done ? 0 : pos < 0 ? 1 : pos / io.split_keys + 1;
    if (ns > io.splits) ns = io.splits;
    float m = kNegBig, z = 0.f;
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
    auto add = [&](float pm, float pz, f32x4 po) {
      const float mn = fmaxf(m, pm);
      const float a = fast_exp2(m - mn), e = fast_exp2(pm - mn);
      o = o * a + po * e;
      z = z * a + pz * e;
      m = mn;
    };
#pragma unroll 4
    for (int s = sub; s < ns; s += SUB) {
      const long long at = s * nrows + row;
      const float2 ml = *reinterpret_cast<const float2*>(io.part_ml + 2 * at);
      add(ml.x, ml.y, d < c.D ? ld4(io.part_o + at * c.D + d) : f32x4{0.f, 0.f, 0.f, 0.f});
    }
    if constexpr (SUB > 1) {
#pragma unroll
      for (int x = kQuads; x < 64; x <<= 1) {
        const float pm = __shfl_xor(m, x), pz = __shfl_xor(z, x);
        f32x4 po;
#pragma unroll
        for (int y = 0; y < 4; ++y) po[y] = __shfl_xor(o[y], x);
        add(pm, pz, po);
      }
    }
    if constexpr (SUB > kWave) {
      const int wave = threadIdx.x >> 6;
      if ((threadIdx.x & 63) < kQuads) st4(&join[wave][d], o);
      if ((threadIdx.x & 63) == 0) {
        join[wave][DT] = m;
        join[wave][DT + 1] = z;
      }
      __syncthreads();
      m = kNegBig;
      z = 0.f;
      o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; ++w) add(join[w][DT], join[w][DT + 1], ld4(&join[w][d]));
      __syncthreads();
    }
    if (done || sub > 0) continue;
    const float inv = z == 0.f ? 0.f : 1.0f / z;
    if (d < c.D)
      st4(static_cast<E*>(io.out) + (long long)(sp.t0 + t) * io.o_ts + (long long)head * io.o_hs + d, o * inv);
    if (io.stats && d == 0) {
      io.stats[2 * row] = m;
      io.stats[2 * row + 1] = inv;
    }
  }
}

// sums[b][h][key] += sum over the sequence's rows of their weight of key.  A wave
// keeps one tile's K rows and walks the rows that see any of its keys; a sum is
// added to by one lane alone, in a fixed order.
template <class E, int DT>
__global__ __launch_bounds__(256) void ca_paged_sums_kernel(PagedAttnIO io) {
  const PagedCache& c = io.c;
  const int lane = threadIdx.x & 63, i16 = lane & 15, G4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int slices = c.batch * c.heads;
  const int slice = blockIdx.x % slices, part = blockIdx.x / slices;
  const int b = slice / c.heads, h = slice - b * c.heads;
  const SeqSpan sp = seq_span(c, b, io.tokens);
  const int rows = sp.n * io.group;
  if (rows == 0) return;
  const int* table = c.table + (long long)b * c.table_stride;
  const E* kh = static_cast<const E*>(c.k) + (long long)h * c.head_stride;
  float* sums = io.sums + (long long)b * io.sums_bs + (long long)h * io.sums_hs;
  const int len = sp.len < io.sums_len ? sp.len : io.sums_len;
  const int parts = gridDim.x / slices;
  for (int first = (part * 4 + wave) * kOwned; first < len; first += parts * 4 * kOwned) {
    const int key = first - 1;  // key of slot 0
    float acc[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) acc[r] = 0.f;
    // first row that sees key + 1
    int t0 = key + 1 - (sp.len - sp.n);
    if (t0 < 0) t0 = 0;
    int r0 = t0 * io.group / 16 * 16;
    RowRef ref[2];
    bool bad = false;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      int at = key + k_slot(x);
      at = at < 0 ? 0 : at > sp.len - 1 ? sp.len - 1 : at;
      const int idx = page_of(c.div, at), page = table[idx];
      bad = bad || (unsigned)page >= (unsigned)c.num_pages;
      ref[x] = RowRef{page_in(c, page), at - idx * (int)c.div.size};
    }
    struct Row {
      Rows<E, DT> q;
      float m, inv;
    };
    auto load_row = [&](int r) {
      Row o;
      o.q = load_rows<E, DT>(io, sp, h, r + i16);
      o.m = o.q.row >= 0 ? io.stats[2 * o.q.row] : 0.f;
      o.inv = o.q.row >= 0 ? io.stats[2 * o.q.row + 1] : 0.f;
      return o;
    };
    Row next = load_row(r0);
    const int slot = 8 * G4 + i16;
    const bool mine = i16 < 8 && slot > 0 && slot < 31 && key + slot < len;
    const float before = mine ? sums[key + slot] : 0.f;
    KRows<E, DT> kr;
    load_k<E, DT>(c, kh, ref, kr);
    for (; r0 < rows; r0 += 16) {
      const Row row = next;
      if (r0 + 16 < rows) next = load_row(r0 + 16);
      const Rows<E, DT>& R = row.q;
      float s[8], w[8];
      tile_products<E, DT>(kr, R, s);
#pragma unroll
      for (int r = 0; r < 8; ++r) s[r] = fmaf(s[r], R.scale, -row.m - kShareShift);
      const int pos_min = sp.len - sp.n + r0 / io.group, key0 = key + 8 * G4;
      if (key < 0 || key + 31 > pos_min || r0 + 16 > rows) {
        tile_weights<true>(s, key0, R.pos, w);
        // a row's NaN stays out of the keys it does not see
#pragma unroll
        for (int r = 0; r < 8; ++r) acc[r] += key0 + r <= R.pos ? w[r] * row.inv : 0.f;
      } else {
        tile_weights<false>(s, key0, R.pos, w);
#pragma unroll
        for (int r = 0; r < 8; ++r) acc[r] += w[r] * row.inv;
      }
    }
    if (wave_any(bad)) {
#pragma unroll
      for (int r = 0; r < 8; ++r) acc[r] = nan_value();
    }
    // over the 16 lanes of a row; lane r < 8 keeps slot 8 G4 + r
    float total = 0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      float x = acc[r];
      x += row_rotated<8>(x);
      x += row_rotated<4>(x);
      x += row_rotated<2>(x);
      x += row_rotated<1>(x);
      total = i16 == r ? x : total;
    }
    if (mine) sums[key + slot] = before + total;
  }
}

template <class E, int DT, bool PAGES>
hipError_t run_attention(const PagedAttnIO& io, hipStream_t s) {
  const dim3 grid((unsigned)((long long)io.c.batch * io.c.heads * io.splits * io.row_tiles));
  if (io.tile_group)
    hipLaunchKernelGGL((ca_paged_few_kernel<E, DT, PAGES>), grid, dim3(256), 0, s, io);
  else if (io.waves == 2) {
    if constexpr (std::is_same<E, float>::value) return hipErrorInvalidValue;  // (not planned)
    else hipLaunchKernelGGL((ca_paged_attention_kernel<E, DT, 2, PAGES>), grid, dim3(128), 0, s, io);
  }
  else if (io.waves == 4)
    hipLaunchKernelGGL((ca_paged_attention_kernel<E, DT, 4, PAGES>), grid, dim3(256), 0, s, io);
  else
    hipLaunchKernelGGL((ca_paged_attention_kernel<E, DT, 8, PAGES>), grid, dim3(512), 0, s, io);
  return hipGetLastError();
}
// Work groups of `parts` for each slice (at least one, at most 2^24 - 1 of 256
// threads in all; the kernels walk what more there is).
unsigned grid_of(long long slices, long long parts) {
  const long long most = ((1ll << 24) - 1) / slices;
  return (unsigned)(slices * std::max<long long>(1, std::min(parts, most)));
}
template <class E, int DT>
hipError_t run_combine(const PagedAttnIO& io, hipStream_t s) {
  const long long slices = (long long)io.c.batch * io.c.heads;
  constexpr int kGroups = 256 / (DT / 4), kWave = kGroups / 4;
  // a group walks at most four splits, a wave's groups eight each
  const int sub = io.splits <= 4 ? 1 : io.splits <= 8 * kWave ? kWave : kGroups;
  const long long rows = (long long)io.tokens * io.group / io.c.batch, each = kGroups / sub;
  const long long per = (rows + each - 1) / each;
  const dim3 grid(grid_of(slices, per < 1024 ? per : 1024)), block(256);
  if (sub == 1) hipLaunchKernelGGL((ca_paged_combine_kernel<E, DT, 1>), grid, block, 0, s, io);
  else if (sub == kWave) hipLaunchKernelGGL((ca_paged_combine_kernel<E, DT, kWave>), grid, block, 0, s, io);
  else hipLaunchKernelGGL((ca_paged_combine_kernel<E, DT, kGroups>), grid, block, 0, s, io);
  return hipGetLastError();
}
template <class E, int DT>
hipError_t run_sums(const PagedAttnIO& io, int max_length, hipStream_t s) {
  const long long slices = (long long)io.c.batch * io.c.heads;
  const long long parts = ((long long)max_length + 4 * kOwned - 1) / (4 * kOwned);
  hipLaunchKernelGGL((ca_paged_sums_kernel<E, DT>), dim3(grid_of(slices, parts)), dim3(256), 0, s, io);
  return hipGetLastError();
}

// The least tile width that holds D.
template <class E, class F> hipError_t by_width(int D, F f) {
  if (D <= 32) return f(std::integral_constant<int, 32>{}, (E*)nullptr);
  if (D <= 64) return f(std::integral_constant<int, 64>{}, (E*)nullptr);
  return f(std::integral_constant<int, 128>{}, (E*)nullptr);
}
template <class F> hipError_t by_type(int dtype, int D, F f) {
  if (dtype == CA_DTYPE_F32) return by_width<float>(D, f);
  if (dtype == CA_DTYPE_BF16) return by_width<__bf16>(D, f);
  return by_width<_Float16>(D, f);
}

}  // namespace

hipError_t launch_paged_attention(const PagedAttnIO& io, int dtype, hipStream_t s) {
  return by_type(dtype, io.c.D, [&](auto width, auto* e) {
    typedef std::remove_pointer_t<decltype(e)> E;
    constexpr int kWidth = decltype(width)::value;
    // Pages that tiles (many rows) or their halves (few) never cross; offsets
    // within a tile in 32 bits.  Halves for many rows as well: pages of 16 the same
    // as looked up row by row (fp32 prompts 200 against 202 us), those of 32 and
    // more slower for it (512 tokens over 8192 112 against 125).
    const bool whole = io.c.div.size % (io.tile_group ? 16 : 32) == 0 && io.c.row_stride < 1 << 25;
    return whole ? run_attention<E, kWidth, true>(io, s) : run_attention<E, kWidth, false>(io, s);
  });
}
hipError_t launch_paged_combine(const PagedAttnIO& io, int dtype, hipStream_t s) {
  return by_type(dtype, io.c.D, [&](auto width, auto* e) {
    return run_combine<std::remove_pointer_t<decltype(e)>, decltype(width)::value>(io, s);
  });
}
hipError_t launch_paged_sums(const PagedAttnIO& io, int dtype, int max_length, hipStream_t s) {
  return by_type(dtype, io.c.D, [&](auto width, auto* e) {
    return run_sums<std::remove_pointer_t<decltype(e)>, decltype(width)::value>(io, max_length, s);
  });
}

}  // namespace ca
