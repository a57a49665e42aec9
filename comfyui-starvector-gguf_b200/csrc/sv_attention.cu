// sv_attention.cu -- entry points of the attention over the decoder's cache: argument
// checks, the split of the slots over blocks, workspace layout and launches.
#include <algorithm>
#include <cmath>

#include "../../include/starvector_sampling.h"
#include "sv_attention.h"
#include "sv_record.cuh"

namespace sv {
namespace {

constexpr int kSMs = 148;
constexpr int kMostPrefixSplits = 16;  // that the token kernel joins
constexpr int kMostSlots = 1 << 29;    // sums of two slot numbers stay in 31 bits
// Groups of query rows that the kernel over 4-bit records takes one by one; more go through plain values.  16 units over
// 4097 slots, bfloat16: 63 rows 71 us (four groups); 72 rows 94 us from plain values, 86 us in five groups; 90 rows 95 and
// 101 us, 126 rows 96 and 131 us.  4 x 4 units over 16384 slots: 63 rows 61 us, 72 rows 107 and 72 us, 126 rows 107 and 106 us,
// 189 rows 121 and 152 us.
constexpr int kMostRecordGroups = 4;
constexpr size_t kMostValues = (size_t)96 << 20;  // bytes of plain values of 4-bit records at a time: they stay in L2
constexpr size_t kMostScores = (size_t)256 << 20;  // bytes of scores kept for the accumulated weights

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

int div_up(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// The most slots one row's query tile can see.
int64_t most_slots(int32_t capacity, int32_t window, int32_t sinks, int64_t tile_queries) {
  if (!window) return capacity;
  const int64_t x = (int64_t)window + sinks + tile_queries - 1;
  return x < capacity ? x : capacity;
}

// Splits of the slots among blocks of the f32 kernel (one per SM): one round of blocks
// at most, at least 128 slots each.
int f32_splits(int64_t blocks, int64_t slots) {
  const int64_t want = kSMs / blocks, most = (slots + 127) / 128;
  const int64_t s = want < most ? want : most;
  return (int)(s < 1 ? 1 : s);
}

// The tile kernel's (one block per SM): with blocks of one tile, one round of blocks at
// most, at least four 64-slot steps each.  A block's two halves pay over many steps: 100
// queries over 2048 slots (36 steps) 30.4 us, 35.3 us without; a prefix of 8192 slots in
// seven splits (19 steps) 63.9 us, 62.5 us without.
TileSplit tile_split(int64_t units, int64_t rows_m, int64_t slots, int most_splits) {
  TileSplit x;
  x.tiles = units * div_up(rows_m, 128) <= kSMs ? 1 : 2;
  const int64_t want = kSMs / (units * div_up(rows_m, 128 * x.tiles)), most = (slots + 255) / 256;
  const int64_t s = want < most ? want : most;
  x.splits = (int)(s < 1 ? 1 : (s > most_splits ? most_splits : s));
  x.paired = x.tiles == 1 && slots / x.splits >= 1536;
  return x;
}

// The token kernel (16-bit types, at most 16 query rows per key/value head) or the
// tile kernels.
bool by_token(const AttnArgs& a) { return a.dtype != SV_F32 && (int64_t)a.n * a.group <= kTokenRows; }

struct Plan {
  bool token;
  int p_splits, o_splits, w_splits;
  TileSplit prefix, own;
  size_t counters, o_bytes, ml_bytes, po_bytes, pml_bytes, lse_bytes, score_bytes, weight_bytes;
  size_t total() const { return counters + o_bytes + ml_bytes + po_bytes + pml_bytes + lse_bytes + score_bytes + weight_bytes; }
};

Plan make_plan(const AttnArgs& a) {
  Plan p = {};
  const int64_t nG = (int64_t)a.n * a.group, all = a.rows * a.kv_heads * nG;
  const int64_t units = (int64_t)a.rows * a.kv_heads;
  // One size whatever the shape: a workspace may serve calls of other shapes in turn,
  // and their partial results must not reach what this call counts in.
  p.counters = SV_ATTENTION_ZERO_BYTES;
  p.token = by_token(a);
  const bool f32 = a.dtype == SV_F32;
  if (a.prefix) {
    const int64_t m = a.rows * nG;
    if (f32) {
      p.p_splits = f32_splits(a.kv_heads * div_up(m, 16), a.prefix);
    } else {
      p.prefix = tile_split(a.kv_heads, m, a.prefix, p.token ? kMostPrefixSplits : kSMs);
      p.p_splits = p.prefix.splits;
    }
    p.po_bytes = up256(p.p_splits * all * a.dim * 4);
    p.pml_bytes = up256(p.p_splits * all * 8);
  }
  if (p.token) {
    p.o_bytes = up256((size_t)2 * kTokenBlocks * 16 * a.dim * 4);
    p.ml_bytes = up256((size_t)2 * kTokenBlocks * 16 * 8);
    p.score_bytes = a.weights ? up256(all * a.capacity * 4) : 0;
    if (p.score_bytes > kMostScores) p.score_bytes = 0;  // the weights take a second product instead
  } else {
    if (f32) {
      const int64_t slots = most_slots(a.capacity, a.window, a.sinks, div_up(16, a.group));
      p.o_splits = f32_splits(units * div_up(nG, 16), slots);
    } else {
      p.own = tile_split(units, nG, most_slots(a.capacity, a.window, a.sinks, div_up(128, a.group)), kSMs);
      if (a.k_low && a.dim > 64) p.own.paired = false;  // its ring holds three steps
      p.o_splits = p.own.splits;
    }
    if (!a.prefix && p.o_splits == 1) p.o_splits = 0;
    p.o_bytes = up256(p.o_splits * all * a.dim * 4);
    p.ml_bytes = up256(p.o_splits * all * 8);
  }
  p.lse_bytes = a.weights ? up256(all * 4) : 0;
  p.w_splits = 1;
  if (a.weights && !p.score_bytes) {  // about four blocks per SM, at least 64 query rows each
    const int64_t want = 4 * kSMs / (units * div_up(a.capacity, f32 ? 64 : 128)), most = div_up(nG, 64);
    const int64_t s = want < most ? want : most;
    p.w_splits = (int)(s < 1 ? 1 : s);
    p.weight_bytes = p.w_splits > 1 ? up256(p.w_splits * units * a.capacity * 4) : 0;
  }
  return p;
}

int check_shapes(const AttnArgs& a) {
  if (a.dtype != SV_F32 && a.dtype != SV_F16 && a.dtype != SV_BF16) return SV_E_DTYPE;
  if (a.rows < 1 || a.n < 1 || a.heads < 1 || a.kv_heads < 1 || a.heads % a.kv_heads || a.capacity < 1)
    return SV_E_SHAPE;
  if (a.dim < 8 || a.dim > kAttnMaxDim || a.dim % 8) return SV_E_SHAPE;
  if ((int64_t)a.rows * a.kv_heads > 65535 || (int64_t)a.rows * a.n * a.heads > (int64_t)1 << 30) return SV_E_SHAPE;
  if (a.window < 0 || a.sinks < 0 || a.capacity > kMostSlots || a.prefix > kMostSlots) return SV_E_SHAPE;
  // The token kernel counts chunks of 64 slots in 31 bits (a cache of broadcast rows could exceed them).
  if ((int64_t)a.rows * a.kv_heads * (a.capacity / 64 + 3) >= (int64_t)1 << 31) return SV_E_SHAPE;
  return SV_OK;
}

int check_pointers(const AttnArgs& a, double scale) {
  if (!a.q || !a.k || !a.v || !a.out || (a.prefix && (!a.pk || !a.pv))) return SV_E_ARG;
  if (!std::isfinite(scale)) return SV_E_RANGE;
  const int64_t e = a.dtype == SV_F32 ? 4 : 2;
  const int64_t strides[8] = {a.q_row, a.q_tok, a.q_head, a.kv_row, a.kv_head, a.kv_slot, a.p_head, a.p_slot};
  for (int64_t s : strides)
    if (s < 0 || s * e % 16) return SV_E_ALIGN;
  const void* ptrs[6] = {a.q, a.k, a.v, a.pk, a.pv, a.out};
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) % 16) return SV_E_ALIGN;
  if (a.weights && (a.w_row < 0 || a.w_head < 0)) return SV_E_SHAPE;
  // Rows and heads add to their own words without atomics.
  if (a.weights && !entries_apart<2>(a.capacity, {a.rows, a.kv_heads}, {a.w_row, a.w_head})) return SV_E_SHAPE;
  // One slot for all positions is no cache (and no dimension of a copy).
  if ((a.capacity > 1 && a.kv_slot == 0) || (a.prefix > 1 && a.p_slot == 0)) return SV_E_SHAPE;
  // Outputs take their own queries' place after those have been read, which blocks do apart from
  // one another; other places hold queries still to be read, as all do for the weights' second product.
  const int64_t sizes[3] = {a.rows, a.n, a.heads}, steps[3] = {a.q_row, a.q_tok, a.q_head};
  bool same = a.q == a.out && !a.weights;
  int64_t span = a.dim, packed = a.dim;
  for (int d = 2; d >= 0; --d) {
    same = same && (sizes[d] == 1 || steps[d] == packed);
    packed *= sizes[d];
    span += (sizes[d] - 1) * steps[d];
  }
  const uintptr_t q = reinterpret_cast<uintptr_t>(a.q), out = reinterpret_cast<uintptr_t>(a.out);
  if (!same && out < q + (uintptr_t)(span * e) && q < out + (uintptr_t)(packed * e)) return SV_E_ARG;
  return SV_OK;
}

// The accumulated weights by a second product, from the rows' sums.
int run_weights(const AttnArgs& a, cudaStream_t stream) {
  if ((a.dtype == SV_F32 ? launch_attn_weights(a, stream) : launch_weights16(a, stream)) != cudaSuccess)
    return SV_E_CUDA;
  return a.w_splits > 1 && launch_weights_sum(a, stream) != cudaSuccess ? SV_E_CUDA : SV_OK;
}

int run(AttnArgs& a, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  const Plan p = make_plan(a);
  if (p.total() && (!workspace || workspace_bytes < p.total())) return SV_E_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return SV_E_ALIGN;
  unsigned char* w = static_cast<unsigned char*>(workspace);
  auto take = [&](size_t bytes) {
    unsigned char* at = w;
    w += bytes;
    return bytes ? at : nullptr;
  };
  a.p_splits = p.p_splits;
  a.o_splits = p.o_splits;
  a.w_splits = p.w_splits;
  a.counters = reinterpret_cast<unsigned*>(take(p.counters));
  a.part_o = reinterpret_cast<float*>(take(p.o_bytes));
  a.part_ml = reinterpret_cast<float2*>(take(p.ml_bytes));
  a.prefix_o = reinterpret_cast<float*>(take(p.po_bytes));
  a.prefix_ml = reinterpret_cast<float2*>(take(p.pml_bytes));
  a.lse = reinterpret_cast<float*>(take(p.lse_bytes));
  a.scores = reinterpret_cast<float*>(take(p.score_bytes));
  a.weight_parts = reinterpret_cast<float*>(take(p.weight_bytes));
  const bool f32 = a.dtype == SV_F32;
  if (a.prefix &&
      (f32 ? launch_attn_f32(a, true, stream) : launch_attn_tile(a, true, p.prefix, stream)) != cudaSuccess)
    return SV_E_CUDA;
  if (p.token) {
    if (launch_attn_token(a, kTokenBlocks, stream) != cudaSuccess) return SV_E_CUDA;
    if (a.scores) return launch_scores_weights(a, stream) == cudaSuccess ? SV_OK : SV_E_CUDA;
    return a.weights ? run_weights(a, stream) : SV_OK;
  }
  if (a.status && !f32 && launch_attn_status(a, stream) != cudaSuccess) return SV_E_CUDA;
  if ((f32 ? launch_attn_f32(a, false, stream) : launch_attn_tile(a, false, p.own, stream)) != cudaSuccess)
    return SV_E_CUDA;
  if (p.o_splits && launch_attn_combine(a, stream) != cudaSuccess) return SV_E_CUDA;
  return a.weights ? run_weights(a, stream) : SV_OK;
}

// Sinks that cover the cache, or a window as wide, leave no limit.
void set_window(AttnArgs& a, int32_t window, int32_t sinks) {
  const bool limit = window < a.capacity && sinks < a.capacity;
  a.window = window < 0 || limit ? window : 0;
  a.sinks = sinks < 0 || (limit && window > 0) ? sinks : 0;
}

// How a call over 4-bit records is done: by the kernel that takes them as they are (few query rows), or
// from the plain values of the slots that some query sees, as many cache rows at a time as kMostValues holds (long
// prompts read each value many times: turning it once, 8192 slots of four heads take 8 us, is cheaper than in every
// block that reads it; four more warps in the tile kernel that did so took 926 us for 2048 queries over 16384
// slots, 489 us this way).
struct RecordPlan {
  bool direct;
  RecordRows rows;
  size_t counters, o_bytes, ml_bytes, lse_bytes, score_bytes;  // direct
  int32_t batch;                                               // cache rows at a time (direct: whose scores are kept),
  int32_t heads;                                               // direct: key/value heads at a time; otherwise all:
  int32_t halves, pairs, bf16_pairs;                           // float16 values, the keys' in pairs, in bfloat16 too;
  size_t before, array;                                        // bytes of the attention's own, of the keys or values
  int arrays() const { return 2 + pairs + 2 * bf16_pairs; }
  size_t total() const {
    return direct ? counters + o_bytes + ml_bytes + lse_bytes + score_bytes : before + arrays() * array;
  }
};

RecordPlan record_plan(const AttnArgs& a) {
  RecordPlan p = {};
  const int64_t nG = (int64_t)a.n * a.group, units = (int64_t)a.rows * a.kv_heads;
  p.rows.tiles = nG <= 8 || a.dtype == SV_F32 ? 1 : 2;
  p.rows.groups = div_up(nG, 8 * p.rows.tiles);
  const int64_t chunks = div_up(most_slots(a.capacity, a.window, a.sinks, a.n), 128) + 1;
  p.rows.fits = chunks <= 16 && units * p.rows.groups * chunks <= kTokenBlocks;
  p.counters = SV_ATTENTION_ZERO_BYTES;
  p.o_bytes = up256((size_t)2 * kTokenBlocks * 8 * p.rows.tiles * record_dims(a.dim) * 4);
  p.ml_bytes = up256((size_t)2 * kTokenBlocks * 8 * p.rows.tiles * 8);
  // A unit's counter each, and chunks (of at least 128 slots) counted in 31 bits.
  p.direct = p.rows.groups <= kMostRecordGroups && units * p.rows.groups <= 65536 &&
             units * p.rows.groups * (a.capacity / 128 + 8) < (int64_t)1 << 31;
  p.heads = a.kv_heads;
  if (p.direct) {
    p.batch = a.rows;
    if (a.weights) {  // as many rows, or of one row as many heads, as kMostScores holds
      const int64_t unit = nG * a.capacity * 4, fit = std::max<int64_t>(kMostScores / unit, 1);
      if (fit < units) p.batch = (int32_t)std::max<int64_t>(fit / a.kv_heads, 1);
      p.heads = (int32_t)std::min<int64_t>(fit, a.kv_heads);
      p.lse_bytes = up256((size_t)p.batch * p.heads * nG * 4);
      p.score_bytes = up256((size_t)p.batch * p.heads * unit);
    }
  } else {
    p.halves = a.dtype != SV_F32;
    p.pairs = a.dtype == SV_F16;
    p.bf16_pairs = a.dtype == SV_BF16 && a.weights;  // (the accumulated weights' product takes keys of the queries' type)
    const size_t row = (size_t)a.kv_heads * a.capacity * a.dim * (a.dtype == SV_F32 ? 4 : 2);
    const size_t fit = kMostValues / (p.arrays() * row);
    p.batch = fit >= (size_t)a.rows ? a.rows : fit > 1 ? (int32_t)fit : 1;
    p.array = up256(p.batch * row);
    static const char some = 0;
    AttnArgs b = a;
    b.halves = p.halves;
    b.k_low = p.pairs ? &some : nullptr;
    for (int32_t rows : {p.batch, a.rows % p.batch}) {
      b.rows = rows;
      if (rows) p.before = std::max(p.before, make_plan(b).total());
    }
  }
  return p;
}

AttnArgs base_args(int32_t dtype, int32_t rows, int32_t tokens, int32_t heads, int32_t kv_heads, int32_t head_dim,
                   int32_t capacity) {
  AttnArgs a = {};
  a.dtype = dtype;
  a.rows = rows;
  a.n = tokens;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.group = kv_heads > 0 ? heads / kv_heads : 0;
  a.dim = head_dim;
  a.capacity = capacity;
  return a;
}

}  // namespace
}  // namespace sv

using namespace sv;

extern "C" {

size_t sv_window_attention_workspace_bytes(int32_t dtype, int32_t rows, int32_t tokens, int32_t heads,
                                           int32_t kv_heads, int32_t head_dim, int32_t capacity, int32_t window,
                                           int32_t sinks, int32_t with_weights) {
  AttnArgs a = base_args(dtype, rows, tokens, heads, kv_heads, head_dim, capacity);
  set_window(a, window, sinks);
  if (check_shapes(a)) return 0;
  float dummy;
  a.weights = with_weights ? &dummy : nullptr;
  return make_plan(a).total();
}

int sv_window_attention(const void* q, int32_t dtype, int32_t rows, int32_t tokens, int32_t heads, int32_t kv_heads,
                        int32_t head_dim, int64_t q_stride_row, int64_t q_stride_token, int64_t q_stride_head,
                        const void* keys, const void* values, int32_t capacity, int64_t kv_stride_row,
                        int64_t kv_stride_head, int64_t kv_stride_slot, const int32_t* lengths, const int32_t* starts,
                        int32_t window, int32_t sinks, double scale, float* weights, int64_t weights_stride_row,
                        int64_t weights_stride_head, void* out, void* workspace, size_t workspace_bytes,
                        int32_t* out_status, void* stream) {
  AttnArgs a = base_args(dtype, rows, tokens, heads, kv_heads, head_dim, capacity);
  a.q = q;
  a.q_row = q_stride_row;
  a.q_tok = q_stride_token;
  a.q_head = q_stride_head;
  a.k = keys;
  a.v = values;
  a.kv_row = kv_stride_row;
  a.kv_head = kv_stride_head;
  a.kv_slot = kv_stride_slot;
  a.lengths = lengths;
  a.starts = starts;
  set_window(a, window, sinks);
  a.scale = (float)(scale * 1.4426950408889634);
  a.weights = weights;
  a.w_row = weights_stride_row;
  a.w_head = weights_stride_head;
  a.out = out;
  a.status = out_status;
  int rc = check_shapes(a);
  if (!rc) rc = check_pointers(a, scale);
  return rc ? rc : run(a, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

size_t sv_quantized_attention_workspace_bytes(int32_t dtype, int32_t rows, int32_t tokens, int32_t heads,
                                              int32_t kv_heads, int32_t head_dim, int32_t capacity, int32_t window,
                                              int32_t sinks, int32_t with_weights) {
  AttnArgs a = base_args(dtype, rows, tokens, heads, kv_heads, head_dim, capacity);
  set_window(a, window, sinks);
  if (check_shapes(a)) return 0;
  float dummy;
  a.weights = with_weights ? &dummy : nullptr;
  return record_plan(a).total();
}

int sv_quantized_attention(const void* q, int32_t dtype, int32_t rows, int32_t tokens, int32_t heads, int32_t kv_heads,
                           int32_t head_dim, int64_t q_stride_row, int64_t q_stride_token, int64_t q_stride_head,
                           const void* cache_keys, const void* cache_values, int32_t capacity, int64_t cache_stride_row,
                           int64_t cache_stride_head, int64_t cache_stride_slot, const int32_t* lengths,
                           const int32_t* starts, int32_t window, int32_t sinks, double scale, float* weights,
                           int64_t weights_stride_row, int64_t weights_stride_head, void* out, void* workspace,
                           size_t workspace_bytes, int32_t* out_status, void* stream) {
  AttnArgs a = base_args(dtype, rows, tokens, heads, kv_heads, head_dim, capacity);
  a.q = q;
  a.q_row = q_stride_row;
  a.q_tok = q_stride_token;
  a.q_head = q_stride_head;
  a.k = cache_keys;
  a.v = cache_values;
  a.lengths = lengths;
  a.starts = starts;
  set_window(a, window, sinks);
  a.scale = (float)(scale * 1.4426950408889634);
  a.weights = weights;
  a.w_row = weights_stride_row;
  a.w_head = weights_stride_head;
  a.out = out;
  a.status = out_status;
  int rc = check_shapes(a);
  if (rc) return rc;
  if (cache_stride_row < 0 || cache_stride_head < 0 || cache_stride_slot < 0 || (capacity > 1 && cache_stride_slot == 0))
    return SV_E_SHAPE;
  if (cache_stride_row % 16 || cache_stride_head % 16 || cache_stride_slot % 16) return SV_E_ALIGN;
  const RecordPlan p = record_plan(a);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  unsigned char* w = static_cast<unsigned char*>(workspace);
  if (p.direct) {
    // The queries' and the output's checks; the records' strides are bytes.
    a.kv_row = cache_stride_row;
    a.kv_head = cache_stride_head;
    a.kv_slot = cache_stride_slot;
  } else {
    a.kv_slot = head_dim;
    a.kv_head = (int64_t)capacity * head_dim;
    a.kv_row = kv_heads * a.kv_head;
  }
  rc = check_pointers(a, scale);
  if (rc) return rc;
  if (!workspace || workspace_bytes < p.total()) return SV_E_WORKSPACE;
  // The call's rows from r on, and key/value heads from h on (of records as they are).
  const auto rows_from = [&](AttnArgs& b, int32_t r, int32_t h) {
    const int64_t e = dtype == SV_F32 ? 4 : 2, head = (int64_t)h * a.group;
    b.q = static_cast<const unsigned char*>(q) + (r * q_stride_row + head * q_stride_head) * e;
    b.out = static_cast<unsigned char*>(out) + ((int64_t)r * tokens * heads + head) * head_dim * e;
    if (p.direct) {
      b.k = static_cast<const unsigned char*>(cache_keys) + r * cache_stride_row + h * cache_stride_head;
      b.v = static_cast<const unsigned char*>(cache_values) + r * cache_stride_row + h * cache_stride_head;
    }
    b.lengths = lengths ? lengths + r : nullptr;
    b.starts = starts ? starts + r : nullptr;
    b.status = out_status ? out_status + r : nullptr;
    b.weights = weights ? weights + r * weights_stride_row + h * weights_stride_head : nullptr;
  };
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return SV_E_ALIGN;
  if (p.direct) {
    auto take = [&](size_t bytes) {
      unsigned char* at = w;
      w += bytes;
      return bytes ? at : nullptr;
    };
    a.counters = reinterpret_cast<unsigned*>(take(p.counters));
    a.part_o = reinterpret_cast<float*>(take(p.o_bytes));
    a.part_ml = reinterpret_cast<float2*>(take(p.ml_bytes));
    a.lse = reinterpret_cast<float*>(take(p.lse_bytes));
    a.scores = reinterpret_cast<float*>(take(p.score_bytes));
    for (int32_t r = 0; r < rows; r += p.batch)
      for (int32_t h = 0; h < kv_heads; h += p.heads) {
        AttnArgs b = a;
        b.rows = std::min(p.batch, rows - r);
        b.kv_heads = std::min(p.heads, kv_heads - h);
        rows_from(b, r, h);
        if (launch_attn_record(b, p.rows, s) != cudaSuccess) return SV_E_CUDA;
        if (b.weights && launch_scores_weights(b, s) != cudaSuccess) return SV_E_CUDA;
      }
    return SV_OK;
  }
  ReadArgs x = {};
  x.row = cache_stride_row;
  x.head = cache_stride_head;
  x.slot = cache_stride_slot;
  a.k = x.out[0] = w + p.before;
  a.v = x.out[1] = w + p.before + p.array;
  a.halves = p.halves;
  a.k_low = x.low = p.pairs ? w + p.before + 2 * p.array : nullptr;
  if (weights && p.halves) {
    a.w_k = p.pairs ? a.k : w + p.before + 2 * p.array;
    a.w_low = p.pairs ? a.k_low : w + p.before + 3 * p.array;
  }
  x.dtype = p.halves ? SV_F16 : dtype;
  x.kv_heads = kv_heads;
  x.dim = head_dim;
  x.capacity = x.tokens = capacity;
  x.seen = tokens;
  x.window = a.window;
  x.sinks = a.sinks;
  for (int32_t r = 0; r < rows; r += p.batch) {
    AttnArgs b = a;
    x.rows = b.rows = std::min(p.batch, rows - r);
    x.cache[0] = static_cast<const unsigned char*>(cache_keys) + r * cache_stride_row;
    x.cache[1] = static_cast<const unsigned char*>(cache_values) + r * cache_stride_row;
    rows_from(b, r, 0);
    x.lengths = b.lengths;
    x.starts = b.starts;
    if (launch_read_records(x, s) != cudaSuccess) return SV_E_CUDA;
    if (p.bf16_pairs) {
      ReadArgs z = x;
      z.dtype = SV_BF16;
      z.cache[1] = nullptr;
      z.out[0] = const_cast<void*>(a.w_k);
      z.out[1] = nullptr;
      z.low = const_cast<void*>(a.w_low);
      if (launch_read_records(z, s) != cudaSuccess) return SV_E_CUDA;
    }
    rc = run(b, workspace, p.before, s);
    if (rc) return rc;
  }
  return SV_OK;
}

size_t sv_prefix_attention_workspace_bytes(int32_t dtype, int32_t rows, int32_t tokens, int32_t heads,
                                           int32_t kv_heads, int32_t head_dim, int32_t prefix_length,
                                           int32_t capacity) {
  AttnArgs a = base_args(dtype, rows, tokens, heads, kv_heads, head_dim, capacity);
  a.prefix = prefix_length;
  if (prefix_length < 0 || check_shapes(a)) return 0;
  return make_plan(a).total();
}

int sv_prefix_attention(const void* q, int32_t dtype, int32_t rows, int32_t tokens, int32_t heads, int32_t kv_heads,
                        int32_t head_dim, int64_t q_stride_row, int64_t q_stride_token, int64_t q_stride_head,
                        const void* prefix_keys, const void* prefix_values, int32_t prefix_length,
                        int64_t prefix_stride_head, int64_t prefix_stride_slot, const void* keys, const void* values,
                        int32_t capacity, int64_t kv_stride_row, int64_t kv_stride_head, int64_t kv_stride_slot,
                        const int32_t* lengths, double scale, void* out, void* workspace, size_t workspace_bytes,
                        int32_t* out_status, void* stream) {
  AttnArgs a = base_args(dtype, rows, tokens, heads, kv_heads, head_dim, capacity);
  a.q = q;
  a.q_row = q_stride_row;
  a.q_tok = q_stride_token;
  a.q_head = q_stride_head;
  a.pk = prefix_keys;
  a.pv = prefix_values;
  a.prefix = prefix_length;
  a.p_head = prefix_stride_head;
  a.p_slot = prefix_stride_slot;
  a.k = keys;
  a.v = values;
  a.kv_row = kv_stride_row;
  a.kv_head = kv_stride_head;
  a.kv_slot = kv_stride_slot;
  a.lengths = lengths;
  a.scale = (float)(scale * 1.4426950408889634);
  a.out = out;
  a.status = out_status;
  if (prefix_length < 0) return SV_E_SHAPE;
  int rc = check_shapes(a);
  if (!rc) rc = check_pointers(a, scale);
  return rc ? rc : run(a, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
