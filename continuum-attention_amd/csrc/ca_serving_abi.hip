// C ABI of the generation operators: attention over a paged cache, eviction from
// it, rotary positions, 4-bit products.  Declarations:
// include/continuum_attention_amd.h.
#include <stdint.h>

#include <algorithm>
#include <new>
#include <vector>

#include "ca_evict.h"
#include "ca_int4.h"
#include "ca_paged.h"
#include "ca_rotary.h"

namespace {

using ca::set_error;

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
int element_bytes(int dtype) {
  return dtype == CA_DTYPE_F32 ? 4 : dtype == CA_DTYPE_BF16 || dtype == CA_DTYPE_F16 ? 2 : 0;
}
constexpr int kMaxSlots = 1 << 30;  // slots a sequence may have: tile ends stay below 2^31
constexpr int kMaxSlices = 1 << 21;  // (sequence, key head)s: a launch has at most 2^32 - 1 threads

// A cache's numbers and pointers; `op` names the caller.
int check_cache(const char* op, const ca_paged_cache* c, bool starts = true) {
  if (!c) return set_error(CA_ERR_INVALID, "%s: null cache", op);
  const int e = element_bytes(c->dtype);
  if (!e) return set_error(CA_ERR_INVALID, "%s: unknown dtype %d", op, c->dtype);
  if (c->batch <= 0 || c->heads <= 0 || c->tokens < 0 || c->num_pages <= 0 || c->page_size <= 0 ||
      c->pages_per_seq <= 0 || c->head_dim <= 0)
    return set_error(CA_ERR_INVALID,
                     "%s: invalid sizes batch=%d heads=%d tokens=%d num_pages=%d page_size=%d pages_per_seq=%d "
                     "head_dim=%d", op, c->batch, c->heads, c->tokens, c->num_pages, c->page_size,
                     c->pages_per_seq, c->head_dim);
  if (c->head_dim % 8 || c->head_dim > 128)
    return set_error(CA_ERR_UNSUPPORTED, "%s: head dim %d (multiples of 8 up to 128)", op, c->head_dim);
  if ((long long)c->pages_per_seq * c->page_size > kMaxSlots)
    return set_error(CA_ERR_UNSUPPORTED, "%s: %d pages of %d slots per sequence exceed 2^30", op,
                     c->pages_per_seq, c->page_size);
  if (c->table_stride < c->pages_per_seq)
    return set_error(CA_ERR_INVALID, "%s: table stride %lld below %d pages per sequence", op,
                     c->table_stride, c->pages_per_seq);
  if (c->page_stride < 0 || c->head_stride < 0 || c->row_stride < 0)
    return set_error(CA_ERR_INVALID, "%s: negative strides", op);
  if (!c->k || !c->v || !c->table || !c->lengths || (starts && !c->starts))
    return set_error(CA_ERR_INVALID, "%s: null pointer", op);
  if (!aligned(c->table, 4) || !aligned(c->lengths, 4) || !aligned(c->starts, 4))
    return set_error(CA_ERR_INVALID, "%s: table, lengths and starts must be 4-byte aligned", op);
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || c->page_stride * e % 16 || c->head_stride * e % 16 ||
      c->row_stride * e % 16)
    return set_error(CA_ERR_INVALID, "%s: cache rows must be 16-byte aligned", op);
  return CA_OK;
}

ca::PagedCache kernel_cache(const ca_paged_cache& c) {
  ca::PagedCache k;
  k.k = c.k;
  k.v = c.v;
  k.page_stride = c.page_stride;
  k.head_stride = c.head_stride;
  k.row_stride = c.row_stride;
  k.table = c.table;
  k.lengths = c.lengths;
  k.starts = c.starts;
  k.table_stride = c.table_stride;
  k.pages_per_seq = c.pages_per_seq;
  k.num_pages = c.num_pages;
  k.heads = c.heads;
  k.D = c.head_dim;
  k.batch = c.batch;
  k.div = ca::page_div(c.page_size);
  return k;
}

// How the attention's grid is cut.  max_new and max_length only size it: the
// kernels read what is there from the device and walk all of it.
struct AttnPlan {
  int row_tiles, splits, split_keys, row_log, tile_group, waves;
};
// Rows per key head that share a wave's columns.  From nine 16-bit rows on two
// waves of 16 that share V are faster, though one of them is empty (us at 16
// rows, shared columns / two waves: [4,4096,16,64] 34.3 / 31.6, [16,2048,16,64]
// 47.5 / 43.4, [8,4096,8,128] 44.6 / 39.7); fp32, whose limbs take eight times
// the shared memory, stays (47 / 58, 76 / 107, 117 / 157) and takes four waves
// at least (20 rows of [8,4096,8,128] 157 with two, 131 with four).
constexpr int kFewRows = 16;
constexpr int kCus = 256;
constexpr int kMostSplits = 128;

size_t partial_bytes(int splits, int tokens, int heads, int D) {
  return splits > 1 ? (size_t)splits * tokens * heads * (D + 2) * sizeof(float) : 0;
}

// Many rows: the time, in steps of one tile of one work group, that `slots` work
// groups at once take for row tiles of given lengths (in tiles, longest first, each
// `slices` times) cut at `cut`: each item goes to the slot that is free first.  (A
// length is below 2^13 and there are at most 16 items for a slot: a few
// megabytes at the very most.)
int dealt_steps(int cut, const std::vector<int>& lengths, long long slices, long long slots) {
  std::vector<long long> free_at(64, 0);  // slots that become free at each step
  free_at[0] = slots;
  size_t lo = 0, most = 0;
  auto deal = [&](long long n, int steps) {
    while (n > 0) {
      while (free_at[lo] == 0) ++lo;
      const long long k = std::min(n, free_at[lo]);
      const size_t end = lo + steps;
      free_at[lo] -= k;
      if (end >= free_at.size()) free_at.resize(2 * end, 0);
      free_at[end] += k;
      most = std::max(most, end);
      n -= k;
    }
  };
  for (int len : lengths)
    for (int at = 0; at < len; at += cut) deal(slices, std::min(cut, len - at));
  return (int)most;
}

AttnPlan make_plan(int dtype, int batch, int kv_heads, int heads, int D, int tokens, int max_new, int max_length) {
  const int group = heads / kv_heads;
  const long long rows = (long long)std::max(1, std::min(max_new, tokens)) * group;
  const long long slices = (long long)batch * kv_heads;
  const size_t cap = ca_workspace_cap();
  AttnPlan p;
  long long tiles = 1;  // of rows
  int unit;             // keys that a split is a multiple of
  long long splits;
  const bool f32 = dtype == CA_DTYPE_F32;
  if (rows <= (f32 ? kFewRows : kFewRows / 2)) {
    p.row_log = p.waves = 0;
    while ((1 << p.row_log) < rows) ++p.row_log;
    // tiles of keys that share a wave: as many as leave the device two waves on
    // each SIMD
    p.tile_group = kFewRows >> p.row_log;
    const long long key_tiles = std::max(1, (max_length + 31) / 32);
    while (p.tile_group > 1 && slices * ((key_tiles + p.tile_group - 1) / p.tile_group) < 8 * kCus)
      p.tile_group >>= 1;
    unit = 32 * p.tile_group;
    // eight work groups for each CU (ragged lengths leave some empty: 32 tokens
    // over up to 8192 slots 127 us with four, 116 with eight, 122 with 16), one
    // group of tiles at least for each of their waves
    const int units = std::max(1, (max_length + unit - 1) / unit);
    splits = std::min<long long>(8 * kCus / slices, units / 4);
  } else {
    p.row_log = p.tile_group = 0;
    p.waves = rows <= 32 && !f32 ? 2 : rows <= 64 ? 4 : 8;
    const int tile_rows = 16 * p.waves;
    tiles = (rows + tile_rows - 1) / tile_rows;
    unit = 32;
    // By estimated time.  Work groups at once: those whose waves and shared memory
    // fit; a step takes about 2 us per 64 columns with the device full, and a
    // partial row 0.2 ns a column pair to write and read again.
    const int simd_waves = D <= 32 ? 4 : D <= 64 ? 4 : 2;
    long long per_cu = std::max(1, 4 * simd_waves / p.waves);
    if (f32) per_cu = std::min<long long>(per_cu, D <= 32 ? 4 : D <= 64 ? 2 : 1);
    const int key_tiles = std::max(1, (max_length + 31) / 32);
    const int coarse = 1 + key_tiles / 4096;  // key tiles counted as one below
    splits = 1;
    try {
      std::vector<int> lengths;  // of up to 64 row tiles (more are much alike)
      const int shown = (int)std::min<long long>(tiles, 64);
      for (int t = 0; t < shown; ++t) {
        const long long last = std::min<long long>(rows, (tiles - t * tiles / shown) * tile_rows) - 1;
        const long long keys = std::max<long long>(1, max_length - (rows - 1 - last) / group);
        lengths.push_back((int)((keys + 32ll * coarse - 1) / (32 * coarse)));
      }
      const long long copies = slices * tiles / shown;  // work groups per length
      const double step_us = 0.55 * p.waves * per_cu / (simd_waves * 4) * 4 * std::max(1.0, D / 64.0) * (f32 ? 1.7 : 1.0);
      double best = 0;
      // (with 16 work groups for each slot the last ones cost little, cut or not)
      if (slices * tiles < 16 * per_cu * kCus)
        for (int s : {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 24, 32, 48, 64}) {
          if (s > 1 && key_tiles / s < 4) break;
          const int cut = (key_tiles + s * coarse - 1) / (s * coarse);
          double us = step_us * coarse * dealt_steps(cut, lengths, copies, per_cu * kCus);
          if (s > 1) {
            double parts = 0;  // row tiles that one split covers write none
            for (int len : lengths) parts += len > cut ? (len + cut - 1) / cut : 0;
            us += 4 + parts / shown * slices * rows * D * 2.5e-4 / 64;
          }
          if (s == 1 || us < best) {
            best = us;
            splits = s;
          }
        }
    } catch (const std::bad_alloc&) {
      splits = 1;  // no memory for the estimate
    }
  }
  const int units = std::max(1, (max_length + unit - 1) / unit);
  splits = std::max<long long>(1, std::min<long long>({splits, kMostSplits, units}));
  while (splits > 1 && cap && partial_bytes((int)splits, tokens, heads, D) > cap) --splits;
  const int per = (units + (int)splits - 1) / (int)splits;
  p.splits = (units + per - 1) / per;
  p.split_keys = per * unit;
  // at most 2^32 - 1 threads, 512 in a work group; each walks the row tiles behind its first
  p.row_tiles = (int)std::max<long long>(1, std::min<long long>(tiles, ((1ll << 23) - 1) / (slices * p.splits)));
  return p;
}

// The last plans of this thread: a decoder asks for the same ones layer after layer.
AttnPlan attn_plan(int dtype, int batch, int kv_heads, int heads, int D, int tokens, int max_new, int max_length) {
  struct Entry {
    long long key[9];
    AttnPlan plan;
  };
  static thread_local Entry kept[16];
  static thread_local unsigned used = 0;
  const long long key[9] = {dtype, batch, kv_heads, heads, D, tokens, max_new, max_length, (long long)ca_workspace_cap()};
  for (unsigned i = 0; i < std::min(used, 16u); ++i)
    if (std::equal(key, key + 9, kept[i].key)) return kept[i].plan;
  const AttnPlan plan = make_plan(dtype, batch, kv_heads, heads, D, tokens, max_new, max_length);
  Entry& e = kept[used++ % 16];
  e.plan = plan;
  std::copy(key, key + 9, e.key);
  return plan;
}
size_t stats_bytes(int tokens, int heads) { return ((size_t)tokens * heads * 2 * sizeof(float) + 255) & ~(size_t)255; }

}  // namespace

extern "C" {

size_t ca_paged_attention_workspace_bytes(int dtype, int batch, int kv_heads, int heads, int head_dim, int tokens,
                                          int max_new, int max_length, int with_sums) {
  if (batch <= 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads || head_dim <= 0 || tokens <= 0 || max_new < 0 ||
      max_length < 0 || max_length > kMaxSlots || (long long)batch * kv_heads > kMaxSlices)
    return 0;
  const AttnPlan p = attn_plan(dtype, batch, kv_heads, heads, head_dim, tokens, max_new, max_length);
  return partial_bytes(p.splits, tokens, heads, head_dim) + (with_sums ? stats_bytes(tokens, heads) : 0);
}

int ca_paged_attention(const ca_paged_cache* cache, const void* q, long long q_token_stride,
                       long long q_head_stride, int heads, const float* log_gain, void* out,
                       long long out_token_stride, long long out_head_stride, float* sums,
                       long long sums_batch_stride, long long sums_head_stride, int sums_len, int max_new,
                       int max_length, void* workspace, size_t workspace_bytes, void* stream) {
  const char* op = "ca_paged_attention";
  int rc = check_cache(op, cache);
  if (rc) return rc;
  if (heads <= 0 || heads % cache->heads)
    return set_error(CA_ERR_INVALID, "%s: %d query heads over %d key heads", op, heads, cache->heads);
  if (cache->tokens == 0) return CA_OK;
  if (!q || !log_gain || !out) return set_error(CA_ERR_INVALID, "%s: null pointer", op);
  const int e = element_bytes(cache->dtype);
  if (!aligned(q, 16) || q_token_stride * e % 16 || q_head_stride * e % 16)
    return set_error(CA_ERR_INVALID, "%s: query rows must be 16-byte aligned", op);
  if (!aligned(out, 16) || out_token_stride * e % 16 || out_head_stride * e % 16)
    return set_error(CA_ERR_INVALID, "%s: output rows must be 16-byte aligned", op);
  if (!aligned(log_gain, 4) || !aligned(sums, 4))
    return set_error(CA_ERR_INVALID, "%s: log_gain and sums must be 4-byte aligned", op);
  if ((long long)cache->tokens * heads * cache->head_dim > (1ll << 31) - 1)
    return set_error(CA_ERR_UNSUPPORTED, "%s: %d tokens of %d heads exceed 2^31 elements", op, cache->tokens, heads);
  if ((long long)cache->batch * cache->heads > kMaxSlices)
    return set_error(CA_ERR_UNSUPPORTED, "%s: %d sequences of %d heads exceed 2^21", op, cache->batch, cache->heads);
  if (max_new < 0 || max_length < 0 || sums_len < 0)
    return set_error(CA_ERR_INVALID, "%s: negative max_new, max_length or sums_len", op);
  max_length = std::min(max_length, cache->pages_per_seq * cache->page_size);
  const size_t need = ca_paged_attention_workspace_bytes(cache->dtype, cache->batch, cache->heads, heads,
                                                         cache->head_dim, cache->tokens, max_new, max_length, sums != nullptr);
  if (need && (!workspace || workspace_bytes < need))
    return set_error(CA_ERR_WORKSPACE, "%s: workspace of %zu bytes required, %zu given", op, need, workspace_bytes);
  if (!aligned(workspace, 16)) return set_error(CA_ERR_INVALID, "%s: workspace must be 16-byte aligned", op);

  const AttnPlan p = attn_plan(cache->dtype, cache->batch, cache->heads, heads, cache->head_dim, cache->tokens, max_new,
                               max_length);
  ca::PagedAttnIO io;
  io.c = kernel_cache(*cache);
  io.q = q;
  io.out = out;
  io.q_ts = q_token_stride;
  io.q_hs = q_head_stride;
  io.o_ts = out_token_stride;
  io.o_hs = out_head_stride;
  io.log_gain = log_gain;
  char* ws = static_cast<char*>(workspace);
  io.stats = nullptr;
  if (sums) {
    io.stats = reinterpret_cast<float*>(ws);
    ws += stats_bytes(cache->tokens, heads);
  }
  const long long rows = (long long)cache->tokens * heads;
  io.part_o = reinterpret_cast<float*>(ws);
  io.part_ml = io.part_o + (p.splits > 1 ? p.splits * rows * cache->head_dim : 0);
  io.sums = sums;
  io.sums_bs = sums_batch_stride;
  io.sums_hs = sums_head_stride;
  io.sums_len = sums_len;
  io.tokens = cache->tokens;
  io.Hq = heads;
  io.group = heads / cache->heads;
  io.splits = p.splits;
  io.split_keys = p.split_keys;
  io.row_tiles = p.row_tiles;
  io.row_log = p.row_log;
  io.tile_group = p.tile_group;
  io.waves = p.waves;
  io.tile_rows = p.tile_group ? 1 << p.row_log : 16 * p.waves;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  hipError_t err = ca::launch_paged_attention(io, cache->dtype, s);
  if (err == hipSuccess && p.splits > 1) err = ca::launch_paged_combine(io, cache->dtype, s);
  if (err == hipSuccess && sums) err = ca::launch_paged_sums(io, cache->dtype, max_length, s);
  if (err != hipSuccess) return set_error(CA_ERR_HIP, "%s launch: %s", op, hipGetErrorString(err));
  return CA_OK;
}

int ca_evict(const ca_paged_cache* cache, const float* sums, long long sums_batch_stride,
             long long sums_head_stride, int sums_len, int budget, int sinks, int recent,
             const int* new_table, long long new_table_stride, int* kept, float* new_sums,
             int* new_lengths, void* stream) {
  const char* op = "ca_evict";
  int rc = check_cache(op, cache, false);
  if (rc) return rc;
  if (!sums || !new_table || !kept || !new_sums || !new_lengths) return set_error(CA_ERR_INVALID, "%s: null pointer", op);
  if (!aligned(sums, 4) || !aligned(new_table, 4) || !aligned(kept, 4) || !aligned(new_sums, 4) || !aligned(new_lengths, 4))
    return set_error(CA_ERR_INVALID, "%s: pointers must be 4-byte aligned", op);
  if (budget <= 0 || sinks < 0 || recent < 0 || (long long)sinks + recent > budget)
    return set_error(CA_ERR_INVALID, "%s: budget %d must be positive and hold %d sinks and %d recent slots", op,
                     budget, sinks, recent);
  if (sums_len < 0) return set_error(CA_ERR_INVALID, "%s: negative sums_len", op);
  if (new_table_stride <= 0 || new_table_stride < (budget + (long long)cache->page_size - 1) / cache->page_size)
    return set_error(CA_ERR_INVALID, "%s: %lld new pages of %d slots do not hold %d", op, new_table_stride,
                     cache->page_size, budget);
  if ((long long)cache->batch * cache->heads > kMaxSlices)
    return set_error(CA_ERR_UNSUPPORTED, "%s: %d sequences of %d heads exceed 2^21", op, cache->batch, cache->heads);
  ca::EvictIO io;
  io.c = kernel_cache(*cache);
  io.sums = sums;
  io.sums_bs = sums_batch_stride;
  io.sums_hs = sums_head_stride;
  io.sums_len = sums_len;
  io.budget = budget;
  io.sinks = sinks;
  io.recent = recent;
  io.new_table = new_table;
  io.new_table_stride = new_table_stride;
  io.kept = kept;
  io.new_sums = new_sums;
  io.new_lengths = new_lengths;
  io.esize = element_bytes(cache->dtype);
  io.row_pieces = cache->head_dim * io.esize / 16;
  hipError_t err = ca::launch_evict(io, reinterpret_cast<hipStream_t>(stream));
  if (err != hipSuccess) return set_error(CA_ERR_HIP, "%s launch: %s", op, hipGetErrorString(err));
  return CA_OK;
}

static int rotary_io(const char* op, const ca_rotary* r, bool cached, ca::RotaryIO& io) {
  if (!r) return set_error(CA_ERR_INVALID, "%s: null argument", op);
  const int e = element_bytes(r->dtype);
  if (!e) return set_error(CA_ERR_INVALID, "%s: unknown dtype %d", op, r->dtype);
  if (r->tokens < 0 || r->q_heads < 0 || r->k_heads < 0 || r->q_heads + (long long)r->k_heads <= 0 || r->head_dim <= 0)
    return set_error(CA_ERR_INVALID, "%s: invalid sizes tokens=%d heads=%d,%d head_dim=%d", op, r->tokens, r->q_heads,
                     r->k_heads, r->head_dim);
  if (r->rotary_dim <= 0 || r->rotary_dim % 2 || r->rotary_dim > r->head_dim || r->head_dim % 2)
    return set_error(CA_ERR_INVALID, "%s: rotary_dim %d of head dim %d (both even)", op, r->rotary_dim, r->head_dim);
  if ((long long)r->tokens * (r->q_heads + 2ll * r->k_heads) * r->head_dim > (1ll << 38))
    return set_error(CA_ERR_UNSUPPORTED, "%s: %d tokens of %d heads exceed 2^38 elements", op, r->tokens,
                     r->q_heads + r->k_heads);
  if (r->tokens == 0) return CA_OK;
  if ((r->q_heads && (!r->q || !r->q_out)) || (r->k_heads && (!r->k || (!cached && !r->k_out))) || !r->positions || !r->turns)
    return set_error(CA_ERR_INVALID, "%s: null pointer", op);
  if (!aligned(r->turns, 8) || !aligned(r->positions, r->positions64 ? 8 : 4) || !aligned(r->q, e) || !aligned(r->k, e) ||
      !aligned(r->q_out, e) || !aligned(r->k_out, e))
    return set_error(CA_ERR_INVALID, "%s: misaligned pointer", op);
  io.q = r->q;
  io.k = r->k;
  io.v = nullptr;
  io.q_out = r->q_out;
  io.k_out = r->k_out;
  io.q_ts = r->q_token_stride;
  io.q_hs = r->q_head_stride;
  io.k_ts = r->k_token_stride;
  io.k_hs = r->k_head_stride;
  io.v_ts = io.v_hs = 0;
  io.qo_ts = r->q_out_token_stride;
  io.qo_hs = r->q_out_head_stride;
  io.ko_ts = r->k_out_token_stride;
  io.ko_hs = r->k_out_head_stride;
  io.positions = r->positions;
  io.turns = r->turns;
  io.magnitude = r->magnitude;
  io.positions64 = r->positions64;
  io.R = r->rotary_dim;
  io.D = r->head_dim;
  io.Hq = r->q_heads;
  io.Hk = r->k_heads;
  io.tokens = r->tokens;
  io.half = r->half;
  io.inverse = r->inverse;
  io.head_chunks = 1;
  auto rows16 = [&](const void* p, long long ts, long long hs) { return aligned(p, 16) && ts * e % 16 == 0 && hs * e % 16 == 0; };
  io.aligned16 = (!io.Hq || (rows16(io.q, io.q_ts, io.q_hs) && rows16(io.q_out, io.qo_ts, io.qo_hs))) &&
                 (!io.Hk || (rows16(io.k, io.k_ts, io.k_hs) && (cached || rows16(io.k_out, io.ko_ts, io.ko_hs))));
  io.c = ca::PagedCache{};
  return CA_OK;
}

int ca_rotary_embedding(const ca_rotary* r, void* stream) {
  const char* op = "ca_rotary_embedding";
  ca::RotaryIO io;
  int rc = rotary_io(op, r, false, io);
  if (rc || r->tokens == 0) return rc;
  hipError_t err = ca::launch_rotary(io, r->dtype, reinterpret_cast<hipStream_t>(stream));
  if (err != hipSuccess) return set_error(CA_ERR_HIP, "%s launch: %s", op, hipGetErrorString(err));
  return CA_OK;
}

int ca_rotary_append(const ca_rotary* r, const void* v, long long v_token_stride, long long v_head_stride,
                     const ca_paged_cache* cache, void* stream) {
  const char* op = "ca_rotary_append";
  ca::RotaryIO io;
  int rc = rotary_io(op, r, true, io);
  if (rc) return rc;
  rc = check_cache(op, cache);
  if (rc) return rc;
  if (cache->dtype != r->dtype || cache->heads != r->k_heads || cache->head_dim != r->head_dim || cache->tokens != r->tokens)
    return set_error(CA_ERR_INVALID, "%s: the cache's dtype, heads, head dim or tokens differ", op);
  if (r->inverse) return set_error(CA_ERR_INVALID, "%s: inverse has no meaning here", op);
  if (r->tokens == 0) return CA_OK;
  const int e = element_bytes(r->dtype);
  if (!v || !aligned(v, e)) return set_error(CA_ERR_INVALID, "%s: null or misaligned values", op);
  io.v = v;
  io.v_ts = v_token_stride;
  io.v_hs = v_head_stride;
  io.aligned16 = io.aligned16 && aligned(v, 16) && v_token_stride * e % 16 == 0 && v_head_stride * e % 16 == 0;
  io.c = kernel_cache(*cache);
  hipError_t err = ca::launch_rotary(io, r->dtype, reinterpret_cast<hipStream_t>(stream));
  if (err != hipSuccess) return set_error(CA_ERR_HIP, "%s launch: %s", op, hipGetErrorString(err));
  return CA_OK;
}

int ca_int4_linear(const void* x, long long x_stride, const unsigned* codes, const void* scales, const void* zeros,
                   void* y, long long y_stride, int dtype, int M, int N, int K, int group, void* stream) {
  const char* op = "ca_int4_linear";
  const int e = element_bytes(dtype);
  if (!e) return set_error(CA_ERR_INVALID, "%s: unknown dtype %d", op, dtype);
  if (M < 0 || N <= 0 || K <= 0) return set_error(CA_ERR_INVALID, "%s: invalid shape M=%d N=%d K=%d", op, M, N, K);
  if (group != 32 && group != 64 && (group <= 0 || group % 128))
    return set_error(CA_ERR_UNSUPPORTED, "%s: groups of %d columns (32, 64 or a multiple of 128)", op, group);
  if ((long long)N * ((K + 127) / 128 * 128ll) > (1ll << 38) || M > (1 << 19) || K > (1 << 30) || N > (1 << 26))
    return set_error(CA_ERR_UNSUPPORTED, "%s: M=%d N=%d K=%d too large", op, M, N, K);
  if (x_stride < K || y_stride < N) return set_error(CA_ERR_INVALID, "%s: row strides below the rows' lengths", op);
  if (M == 0) return CA_OK;
  if (!x || !codes || !scales || !y) return set_error(CA_ERR_INVALID, "%s: null pointer", op);
  if (!aligned(codes, 16) || !aligned(x, e) || !aligned(scales, 16) || !aligned(zeros, 16) || !aligned(y, e))
    return set_error(CA_ERR_INVALID, "%s: misaligned pointer", op);
  ca::Int4IO io;
  io.x = x;
  io.codes = codes;
  io.scales = scales;
  io.zeros = zeros;
  io.y = y;
  io.x_rs = x_stride;
  io.y_rs = y_stride;
  io.M = M;
  io.N = N;
  io.K = K;
  io.group = group;
  io.x_aligned = aligned(x, 16) && x_stride * e % 16 == 0;
  hipError_t err = ca::launch_int4(io, dtype, reinterpret_cast<hipStream_t>(stream));
  if (err != hipSuccess) return set_error(CA_ERR_HIP, "%s launch: %s", op, hipGetErrorString(err));
  return CA_OK;
}

}  // extern "C"
