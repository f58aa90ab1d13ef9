// Continuum Attention of new tokens over a paged key/value cache (gfx950).
//
// A sequence of cached length L (its n new tokens included) has its query t at
// slot p = L - n + t, which sees keys 0..p with the operator's weights: the
// scores are linear between neighbouring slots, each key takes the integral of
// e^score against its hat function, keys 0 and p half a token more (segment
// math in ca_common.h).  The rows of one key head are its new tokens times the
// query heads that share it, r = t * group + g.
//
// Tiles.  A wave holds 16 rows and walks tiles of 32 key slots, of which it
// owns the middle 30: slots 0 and 31 are the neighbours whose segments reach
// into the tile.  So a tile depends on no other one but for the running
// maximum, and keys can be cut anywhere (between waves, work groups, the pages
// of the cache); 6.7% of the work is done twice for it.  The alternative, tiles
// that carry a score and a share from the one before as the forward kernels do,
// would need a product of its own at every cut.
//
// Products on 16x16 matrix instructions.  S^T = K Q^T: the keys' rows are dealt
// so that lane row G = lane / 16 holds slots 8G .. 8G + 7 of query lane % 16; K
// comes straight from memory into operand registers (a row's D values are dealt
// to the four lane rows in quarters, the queries' alike, so that a lane reads
// consecutive bytes).  O^T += V^T W^T takes the lane's own weights as the other
// operand; V passes through shared memory, where it is read transposed.  16-bit
// operands are exact in the 16-bit instructions; the weights go as two 16-bit
// limbs (relative error 2^-17 in bf16, 2^-20 in fp16, against half a step of
// 2^-9 and 2^-12 that the output's rounding makes).  fp32 operands take the fp32
// instruction: the limb products of the training kernels cost as much time
// once each wave has to split what it reads.
//
// Two shapes of a work group of four waves: up to 16 rows per key head (single
// tokens) all waves hold the same rows and take tiles in turn, each with V of
// its own; more rows are dealt to the waves, which share V.
#include "ca_paged.h"

namespace ca {

namespace {

constexpr int kOwned = 30;  // keys a tile owns

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
__device__ __forceinline__ RowRef row_ref(const PagedCache& c, const int* table, int key, int last) {
  key = key < 0 ? 0 : key > last ? last : key;
  const int idx = page_of(c.div, key);
  return RowRef{table[idx], key - idx * (int)c.div.size};
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
__device__ __forceinline__ void tile_products(const KRows<E, DT>& kr, const Rows<E, DT>& R, float (&s)[8]) {
  typedef Tile<E, DT> P;
  f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
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
#pragma unroll
  for (int r = 0; r < 8; ++r) s[r] = acc[r >> 2][r & 3];
}

// Weights of the lane's eight slots from their scores relative to the row's
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

// O^T += V^T W^T over the tile's 32 slots; vs: the tile's V rows.  FINITE:
// without the values that are not finite.
template <class E, int DT, bool FINITE>
__device__ __forceinline__ void add_values(Running<DT>& st, const E* vs, const float (&w)[8]) {
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
    u32x4 hi, lo;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const float a = w[2 * p], b = w[2 * p + 1];
      if constexpr (std::is_same<E, __bf16>::value) {
        unsigned x[3];
        split_pair_limbs<2>(a, b, x);
        hi[p] = x[0];
        lo[p] = x[1];
      } else {
        typedef __fp16 h2 __attribute__((ext_vector_type(2)));
        const h2 h = __builtin_amdgcn_cvt_pkrtz(a, b);
        const h2 l = __builtin_amdgcn_cvt_pkrtz(a - (float)h[0], b - (float)h[1]);
        hi[p] = __builtin_bit_cast(unsigned, h);
        lo[p] = __builtin_bit_cast(unsigned, l);
      }
    }
    // transposed reads: see lds_read_tr8
    const __bf16* base = reinterpret_cast<const __bf16*>(vs) + (8 * G4 + (i >> 2)) * P::kRow + 4 * (i & 3);
#pragma unroll
    for (int b = 0; b < DT / 16; ++b) {
      u32x4 a = __builtin_bit_cast(u32x4, lds_read_tr8(base + 16 * b, base + 4 * P::kRow + 16 * b));
      if (FINITE) a = finite_part<E>(a);
      st.o[b] = mfma16_of(a, lo, st.o[b], (const E*)nullptr);
      st.o[b] = mfma16_of(a, hi, st.o[b], (const E*)nullptr);
    }
  }
}
// The values that are not finite, key by key, into the rows that see them: in a
// tile that some row sees only in part, a product with their zero weights would
// carry them into rows that must not read them.  Those rows' sums stay as they
// would be with any other values there, bit for bit.
template <class E, int DT>
__device__ __forceinline__ void add_values_seen(Running<DT>& st, const E* vs, const float (&w)[8], int tile_key,
                                                int pos) {
  typedef Tile<E, DT> P;
  const int lane = threadIdx.x & 63, i = lane & 15, G4 = lane >> 4;
#pragma unroll
  for (int r = 0; r < 8; ++r)
    for (int g = 0; g < 4; ++g) {
      const int slot = 8 * g + r;
      const float x = __shfl(w[r], 16 * g + i);
      const bool seen = slot > 0 && slot < 31 && tile_key + slot <= pos;
#pragma unroll
      for (int b = 0; b < DT / 16; ++b) {
        const f32x4 v = ld4(vs + slot * P::kRow + 16 * b + 4 * G4);
#pragma unroll
        for (int e = 0; e < 4; ++e) st.o[b][e] += seen && !is_finite(v[e]) ? x * v[e] : 0.f;
      }
    }
}

__device__ __forceinline__ float nan_value() { return __int_as_float(0x7fc00000); }

// Is a page number of slots [first, last] outside the cache?  (All threads of
// the work group call it.)
__device__ __forceinline__ bool bad_pages(const PagedCache& c, const int* table, int first, int last) {
  bool bad = false;
  const int end = page_of(c.div, last);
  for (int i = page_of(c.div, first) + (int)threadIdx.x; i <= end; i += (int)blockDim.x)
    bad = bad || (unsigned)table[i] >= (unsigned)c.num_pages;
  return __syncthreads_or(bad);
}

// WR: waves that hold different rows (4), or 1: the four waves hold the same 16
// rows and take tiles in turn.
template <class E, int DT, int WR>
__global__ __launch_bounds__(256) void ca_paged_attention_kernel(PagedAttnIO io) {
  typedef Tile<E, DT> P;
  constexpr int kStage = 64 * WR;                                     // threads that stage a tile of V
  constexpr int kV = (32 * P::kChunks + kStage - 1) / kStage;         // 16-byte loads of each
  constexpr int kBufs = WR == 1 ? 4 : 2;                              // one per wave, or two in turn
  constexpr int kVBytes = kBufs * 32 * P::kRow * (int)sizeof(E);
  constexpr int kJoinBytes = WR == 1 ? 4 * 16 * (DT + 4) * (int)sizeof(float) : 0;
  __shared__ __attribute__((aligned(16))) unsigned char lds[kVBytes > kJoinBytes ? kVBytes : kJoinBytes];
  __shared__ int special[kBufs];  // tile (plus one) whose V holds a value that is not finite

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
  const int tiles = (rows + 16 * WR - 1) / (16 * WR);

  // longest rows first
  for (int back = tile0; back < tiles; back += io.row_tiles) {
    const int row0 = (tiles - 1 - back) * 16 * WR;
    const int last_row = row0 + 16 * WR < rows ? row0 + 16 * WR - 1 : rows - 1;
    const int pos_max = sp.len - sp.n + last_row / io.group;  // last slot any row sees
    const int pos_min = sp.len - sp.n + row0 / io.group;
    const int first = split * io.split_keys;
    if (pos_max < first) {
      if (split > 0) continue;  // nothing here; row_splits() says so to the one who joins
    }
    const int end = split == io.splits - 1 ? pos_max + 1
                    : first + io.split_keys < pos_max + 1 ? first + io.split_keys : pos_max + 1;
    const Rows<E, DT> R = load_rows<E, DT>(io, sp, h, row0 + (WR == 1 ? 0 : 16 * wave) + i16);
    Running<DT> st;
    st.m = kNegBig;
    st.z = 0.f;
#pragma unroll
    for (int x = 0; x < DT / 16; ++x) st.o[x] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (tid < kBufs) special[tid] = 0;
    const int ntiles = end > first ? (end - first + kOwned - 1) / kOwned : 0;
    bool bad = false;
    if (ntiles > 0) {
      const int halo = end <= pos_max ? end : pos_max;
      bad = bad_pages(c, table, first > 0 ? first - 1 : 0, halo);
    } else {
      __syncthreads();
    }
    if (bad) {
      st.m = st.z = nan_value();
    } else {
      constexpr int kStep = WR == 1 ? 4 : 1;  // tiles between a wave's
      const int t_first = WR == 1 ? wave : 0;
      E* vbuf = reinterpret_cast<E*>(lds);
      KRows<E, DT> kr;
      RowRef kref[2], vref[kV];
      u32x4 vreg[kV];
      const int stage_id = WR == 1 ? lane : tid;
      auto refs = [&](int t) {  // page numbers of tile t's rows
        const int key = first + t * kOwned - 1;
#pragma unroll
        for (int x = 0; x < 2; ++x) kref[x] = row_ref(c, table, key + k_slot(x), pos_max);
#pragma unroll
        for (int x = 0; x < kV; ++x)
          vref[x] = row_ref(c, table, key + (stage_id + x * kStage) / P::kChunks, pos_max);
      };
      auto load_v = [&](int t) {
        const int key = first + t * kOwned - 1;
#pragma unroll
        for (int x = 0; x < kV; ++x) {
          const int u = stage_id + x * kStage, row = u / P::kChunks, d = u % P::kChunks * P::kVec;
          // rows of other tiles and behind the last key stay out: zeros
          const bool mine = row > 0 && row < 31 && key + row < end && d < c.D;
          vreg[x] = mine ? *reinterpret_cast<const u32x4*>(vh + row_at(c, vref[x]) + d) : u32x4{0, 0, 0, 0};
        }
      };
      auto store_v = [&](int t, int buf) {
        const bool look = first + t * kOwned + 30 > pos_min;
#pragma unroll
        for (int x = 0; x < kV; ++x) {
          const int u = stage_id + x * kStage, row = u / P::kChunks, d = u % P::kChunks * P::kVec;
          if ((32 * P::kChunks) % kStage == 0 || row < 32) {
            *reinterpret_cast<u32x4*>(vbuf + (buf * 32 + row) * P::kRow + d) = vreg[x];
            if (look && any_special(vreg[x], (const E*)nullptr)) special[buf] = t + 1;
          }
        }
      };
      auto sync = [&]() {
        if constexpr (WR == 1) wave_lds_sync(); else __syncthreads();
      };
      if (t_first < ntiles) {
        refs(t_first);
        load_k<E, DT>(c, kh, kref, kr);
        load_v(t_first);
        refs(t_first + kStep);
        store_v(t_first, WR == 1 ? wave : 0);
        sync();
      }
      for (int t = t_first; t < ntiles; t += kStep) {
        const int buf = WR == 1 ? wave : t & 1;
        const int key = first + t * kOwned - 1;  // key of slot 0
        float s[8], w[8];
        tile_products<E, DT>(kr, R, s);
        if (t + kStep < ntiles) {
          load_k<E, DT>(c, kh, kref, kr);
          load_v(t + kStep);
          refs(t + 2 * kStep);
        }
        const int key0 = key + 8 * G4;
        const bool mask = key < 0 || key + 31 > pos_min;
        float mt = kNegBig;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          s[r] *= R.scale;
          mt = fmaxf(mt, !mask || (key0 + r >= 0 && key0 + r <= R.pos) ? s[r] : kNegBig);
        }
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
        const float shift = st.m + (kShareShift - weight_octaves<E>());
#pragma unroll
        for (int r = 0; r < 8; ++r) s[r] -= shift;
        if (mask) tile_weights<true>(s, key0, R.pos, w);
        else tile_weights<false>(s, key0, R.pos, w);
#pragma unroll
        for (int r = 0; r < 8; ++r) st.z += w[r];
        const E* vs = vbuf + buf * 32 * P::kRow;
        if (mask && special[buf] == t + 1) {
          add_values<E, DT, true>(st, vs, w);
          add_values_seen<E, DT>(st, vs, w, key, R.pos);
        } else {
          add_values<E, DT, false>(st, vs, w);
        }
        if (t + kStep < ntiles) store_v(t + kStep, WR == 1 ? wave : buf ^ 1);
        sync();
      }
      st.z = rows_sum(st.z);
    }

    const long long nrows = (long long)io.tokens * io.Hq;
    if constexpr (WR == 1) {
      // join the four waves' parts; row_bytes: O, then m and z
      constexpr int kJRow = DT + 4;
      float* join = reinterpret_cast<float*>(lds);
      __syncthreads();
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
      for (int u = tid; u < 16 * kQuads; u += 256) {
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
        if (io.splits == 1) {
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
    } else {
      const float meff = st.m - weight_octaves<E>();
      if (R.row >= 0) {
        if (io.splits == 1) {
          const float inv = st.z == 0.f ? 0.f : 1.0f / st.z;
          const int r = row0 + 16 * wave + i16, t = r / io.group, head = h * io.group + r - t * io.group;
          E* o = static_cast<E*>(io.out) + (long long)(sp.t0 + t) * io.o_ts + (long long)head * io.o_hs;
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
      __syncthreads();
    }
  }
}

// Joins the splits of a row: one wave per row, DT / 4 lanes over its columns and
// the remaining factor of 64 over the splits.
template <class E, int DT>
__global__ __launch_bounds__(256) void ca_paged_combine_kernel(PagedAttnIO io) {
  constexpr int kQuads = DT / 4, kLanes = 64 / kQuads;
  const PagedCache& c = io.c;
  const int slices = c.batch * c.heads;
  const int slice = blockIdx.x % slices, part = blockIdx.x / slices;
  const int b = slice / c.heads, h = slice - b * c.heads;
  const SeqSpan sp = seq_span(c, b, io.tokens);
  const int rows = sp.n * io.group, lane = threadIdx.x & 63;
  const int d = lane % kQuads * 4, sub = lane / kQuads;
  const long long nrows = (long long)io.tokens * io.Hq;
  const int parts = gridDim.x / slices;
  // every work group of the attention kernel wrote the rows of its tile up to
  // the last slot any of them sees: a row's splits are those up to its own slot
  for (int r = part * 4 + (threadIdx.x >> 6); r < rows; r += 4 * parts) {
    const int t = r / io.group, head = h * io.group + r - t * io.group;
    const long long row = (long long)(sp.t0 + t) * io.Hq + head;
    const int pos = sp.len - sp.n + t;
    int ns = pos < 0 ? 1 : pos / io.split_keys + 1;
    if (ns > io.splits) ns = io.splits;
    float m = kNegBig, z = 0.f;
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int s = sub; s < ns; s += kLanes) {
      const long long at = s * nrows + row;
      const float pm = io.part_ml[2 * at], pz = io.part_ml[2 * at + 1];
      const f32x4 po = d < c.D ? ld4(io.part_o + at * c.D + d) : f32x4{0.f, 0.f, 0.f, 0.f};
      const float mn = fmaxf(m, pm);
      const float a = fast_exp2(m - mn), e = fast_exp2(pm - mn);
      o = o * a + po * e;
      z = z * a + pz * e;
      m = mn;
    }
#pragma unroll
    for (int x = kQuads; x < 64; x <<= 1) {
      const float pm = __shfl_xor(m, x), pz = __shfl_xor(z, x);
      const float mn = fmaxf(m, pm);
      const float a = fast_exp2(m - mn), e = fast_exp2(pm - mn);
#pragma unroll
      for (int y = 0; y < 4; ++y) o[y] = o[y] * a + __shfl_xor(o[y], x) * e;
      z = z * a + pz * e;
      m = mn;
    }
    const float inv = z == 0.f ? 0.f : 1.0f / z;
    if (sub == 0 && d < c.D)
      st4(static_cast<E*>(io.out) + (long long)(sp.t0 + t) * io.o_ts + (long long)head * io.o_hs + d, o * inv);
    if (io.stats && lane == 0) {
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
  for (int first = part * 4 * kOwned; first < len; first += parts * 4 * kOwned) {
    const int halo = first + 4 * kOwned < sp.len ? first + 4 * kOwned : sp.len - 1;
    const bool bad = bad_pages(c, table, first > 0 ? first - 1 : 0, halo);
    const int key = first + wave * kOwned - 1;  // key of slot 0
    if (key + 1 >= len) continue;
    float acc[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) acc[r] = bad ? nan_value() : 0.f;
    if (!bad) {
      KRows<E, DT> kr;
      RowRef ref[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) ref[x] = row_ref(c, table, key + k_slot(x), sp.len - 1);
      load_k<E, DT>(c, kh, ref, kr);
      // first row that sees key + 1
      int t0 = key + 1 - (sp.len - sp.n);
      if (t0 < 0) t0 = 0;
      for (int r0 = t0 * io.group / 16 * 16; r0 < rows; r0 += 16) {
        const Rows<E, DT> R = load_rows<E, DT>(io, sp, h, r0 + i16);
        const float m = R.row >= 0 ? io.stats[2 * R.row] : 0.f;
        const float inv = R.row >= 0 ? io.stats[2 * R.row + 1] : 0.f;
        float s[8], w[8];
        tile_products<E, DT>(kr, R, s);
#pragma unroll
        for (int r = 0; r < 8; ++r) s[r] = fmaf(s[r], R.scale, -m - kShareShift);
        const int pos_min = sp.len - sp.n + r0 / io.group, key0 = key + 8 * G4;
        if (key < 0 || key + 31 > pos_min || r0 + 16 > rows) {
          tile_weights<true>(s, key0, R.pos, w);
          // a row's NaN stays out of the keys it does not see
#pragma unroll
          for (int r = 0; r < 8; ++r) acc[r] += key0 + r <= R.pos ? w[r] * inv : 0.f;
        } else {
          tile_weights<false>(s, key0, R.pos, w);
#pragma unroll
          for (int r = 0; r < 8; ++r) acc[r] += w[r] * inv;
        }
      }
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) {
#pragma unroll
      for (int x = 1; x < 16; x <<= 1) acc[r] += __shfl_xor(acc[r], x);
      const int slot = 8 * G4 + r;
      if (i16 == r && slot > 0 && slot < 31 && key + slot < len) sums[key + slot] += acc[r];
    }
  }
}

template <class E, int DT>
hipError_t run_attention(const PagedAttnIO& io, int wave_rows, hipStream_t s) {
  const long long blocks = (long long)io.c.batch * io.c.heads * io.splits * io.row_tiles;
  if (wave_rows == 1)
    hipLaunchKernelGGL((ca_paged_attention_kernel<E, DT, 1>), dim3((unsigned)blocks), dim3(256), 0, s, io);
  else
    hipLaunchKernelGGL((ca_paged_attention_kernel<E, DT, 4>), dim3((unsigned)blocks), dim3(256), 0, s, io);
  return hipGetLastError();
}
template <class E, int DT>
hipError_t run_combine(const PagedAttnIO& io, hipStream_t s) {
  const long long slices = (long long)io.c.batch * io.c.heads;
  const long long per = ((long long)io.tokens * io.group / io.c.batch + 3) / 4;
  const long long parts = per < 1 ? 1 : per > 256 ? 256 : per;
  hipLaunchKernelGGL((ca_paged_combine_kernel<E, DT>), dim3((unsigned)(slices * parts)), dim3(256), 0, s, io);
  return hipGetLastError();
}
template <class E, int DT>
hipError_t run_sums(const PagedAttnIO& io, int max_length, hipStream_t s) {
  const long long slices = (long long)io.c.batch * io.c.heads;
  const long long parts = ((long long)max_length + 4 * kOwned - 1) / (4 * kOwned);
  hipLaunchKernelGGL((ca_paged_sums_kernel<E, DT>), dim3((unsigned)(slices * (parts < 1 ? 1 : parts))),
                     dim3(256), 0, s, io);
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

hipError_t launch_paged_attention(const PagedAttnIO& io, int dtype, int wave_rows, hipStream_t s) {
  return by_type(dtype, io.c.D, [&](auto width, auto* e) {
    return run_attention<std::remove_pointer_t<decltype(e)>, decltype(width)::value>(io, wave_rows, s);
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
