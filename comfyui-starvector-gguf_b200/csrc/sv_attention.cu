// sv_attention.cu -- entry points of the attention over the decoder's cache: argument
// checks, the split of the slots over blocks, workspace layout and launches.
#include <cmath>

#include "../../include/starvector_sampling.h"
#include "sv_attention.h"

namespace sv {
namespace {

constexpr int kSMs = 148;
constexpr int kMostPrefixSplits = 16;  // that the token kernel joins
constexpr int kMostSlots = 1 << 29;    // sums of two slot numbers stay in 31 bits
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
