// sv_attention.h -- launch descriptors of the cache attention kernels, shared by the
// entry points (sv_attention.cu) and the kernel files.
//
// Query rows are packed by key/value head: the n x G rows (query i, head g of the
// group) that read one head's slots are numbered m = i * G + g, so a tile of rows
// loads each slot once for the whole group.  Over the call a row's index is
//   idx = (r * kv_heads + h) * n * G + m.
// Work that is split over the slots leaves, per split and row, an unnormalised f32
// output and its (maximum, sum) in the workspace; the maximum is in units of
// log2 (score * scale * log2 e), so weights are exp2(s - m).
#pragma once
#include <atomic>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace sv {

constexpr int kAttnMaxDim = 128;
constexpr int kTokenRows = 16;     // query rows per key/value head of the token kernel
constexpr int kTokenWarps = 8;     // its warps per block, blocks per SM, blocks
constexpr int kTokenPerSM = 1;
constexpr int kTokenBlocks = 148 * kTokenPerSM;

struct AttnArgs {
  const void* q;
  int64_t q_row, q_tok, q_head;  // strides in elements; head_dim is contiguous
  const void *k, *v;             // the rows' own slots
  int64_t kv_row, kv_head, kv_slot;
  const void *pk, *pv;  // the shared prefix (prefix = 0: none)
  int64_t p_head, p_slot;
  int32_t prefix;
  int32_t dtype, rows, n, heads, kv_heads, group, dim, capacity;
  const int32_t *lengths, *starts;  // per row, may be null (capacity, 0)
  int32_t window, sinks;            // window 0: none
  float scale;                      // scale * log2 e
  float* weights;                   // accumulated attention weights, may be null
  int64_t w_row, w_head;
  void* out;  // [rows, n, heads, dim]
  int32_t* status;
  // workspace
  unsigned* counters;  // zero between calls: [rows * kv_heads], then two per block of the token kernel
  float* part_o;       // own part: [o_splits][idx][dim], or of the token kernel [2 * blocks][16][dim]
  float2* part_ml;     // the same without dim
  float* prefix_o;     // prefix part: [p_splits][prefix_index][dim]
  float2* prefix_ml;
  float* lse;          // [idx], with weights only: log2 of the softmax denominator, maximum included
  float* scores;       // [idx][capacity], with weights in the token kernel only
  float* weight_parts; // [w_splits][rows * kv_heads][capacity], with weights and w_splits > 1
  int32_t p_splits, o_splits;  // o_splits 0: the own part is written directly
  int32_t w_splits;            // of the query rows, for the accumulated weights of calls with many
  const void* k_low;           // with halves and float16 queries: what the keys' rounding left, laid out as they are
  const void *w_k, *w_low;     // with halves and weights: keys of the queries' type and what their rounding left, as above
  int32_t halves;              // keys and values are float16 whatever the queries are (values of a 4-bit cache)
  int32_t test_head;           // test hook: one plus the key/value head whose waits run out
};

// A prefix part's rows are numbered by head first: (h * rows + r) * n * G + m.
__device__ __forceinline__ int64_t prefix_index(const AttnArgs& a, int r, int h, int m) {
  return ((int64_t)h * a.rows + r) * a.n * a.group + m;
}

// The slots that row r's queries can see: queries stand at p = end - n + i, slots
// before `start` (padding in front) are never seen.
struct RowSpan {
  int start, end;
};

__device__ __forceinline__ RowSpan row_span(const AttnArgs& a, int r) {
  int end = a.lengths ? a.lengths[r] : a.capacity;
  end = min(max(end, 0), a.capacity);
  int start = a.starts ? a.starts[r] : 0;
  start = min(max(start, 0), end);
  return {start, end};
}

// First slot of the window of a query at position p.
__device__ __forceinline__ int window_low(const AttnArgs& a, int start, int p) {
  return a.window ? max(start, p - a.window + 1) : start;
}

// Whether the query at p (window from lo) sees slot j of a row that starts at start.
__device__ __forceinline__ bool slot_seen(const AttnArgs& a, int start, int p, int lo, int j) {
  return j <= p && j >= start && (j >= lo || j < start + a.sinks);
}

template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// Eight consecutive elements as floats (16-byte aligned for the 16-bit types, two
// such vectors for float).
__device__ __forceinline__ void load8(const float* p, float* x) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void load8(const __half* p, float* x) {
  const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
  const __half2* h = reinterpret_cast<const __half2*>(&a);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float* x) {
  const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&a);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(h[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

// Whether the entries of a strided array that is written are apart from one another:
// runs of `extent` contiguous elements, D dimensions of `sizes` entries at `strides`.
// From the smallest stride up, each has to step over all that lies within it (layouts
// that interleave dimensions otherwise are refused, apart or not).
template <int D> bool entries_apart(int64_t extent, const int64_t (&sizes)[D], const int64_t (&strides)[D]) {
  bool done[D] = {};
  for (int k = 0; k < D; ++k) {
    int at = -1;
    for (int d = 0; d < D; ++d)
      if (!done[d] && (at < 0 || strides[d] < strides[at])) at = d;
    done[at] = true;
    if (sizes[at] <= 1) continue;  // the stride of one entry means nothing
    if (strides[at] < extent) return false;
    extent += (sizes[at] - 1) * strides[at];
  }
  return true;
}

// Raises a kernel's shared-memory limit, once per device and process.
template <auto Kernel> cudaError_t allow_smem(size_t bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? (uint64_t)1 << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// Programmatic dependent launch: a kernel launched by launch_after may start once every
// block of the kernel before it in the stream has called launch_dependents (or ended); it
// calls wait_before before it uses that kernel's results, and before it ends, so that
// what comes after it in the stream finds both done.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... P, typename... A>
cudaError_t launch_after(bool early, void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem,
                         cudaStream_t stream, A... args) {
  cudaLaunchConfig_t c = {};
  c.gridDim = grid;
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = smem;
  c.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  c.attrs = &attr;
  c.numAttrs = early ? 1 : 0;
  return cudaLaunchKernelEx(&c, kernel, args...);
}

// The query rows [first, last) that share `split` of the sum over those that may see
// slots [j0, j0 + count): under the causal mask none before the first whose position
// reaches j0, under a window none past the last that still has the last of them.
__device__ __forceinline__ void weight_rows(const AttnArgs& a, const RowSpan& sp, int j0, int count, int split,
                                            int& first, int& last) {
  const int nG = a.n * a.group, at = sp.end - a.n;
  const int64_t lo = max(0, j0 - at) * (int64_t)a.group;
  int64_t hi = nG;
  if (a.window && j0 >= sp.start + a.sinks) hi = ((int64_t)j0 + count - 1 + a.window - at) * a.group;
  hi = min((int64_t)nG, max(hi, lo));
  first = (int)(lo + (hi - lo) * split / a.w_splits);
  last = (int)(lo + (hi - lo) * (split + 1) / a.w_splits);
}

// A slot's sum: added to the weights, or left for launch_weights_sum.
__device__ __forceinline__ void add_weight(const AttnArgs& a, int unit, int r, int h, int j, int split, float x) {
  if (a.w_splits > 1)
    a.weight_parts[((int64_t)split * a.rows * a.kv_heads + unit) * a.capacity + j] = x;
  else
    a.weights[r * a.w_row + h * a.w_head + j] += x;
}

cudaError_t launch_weights_sum(const AttnArgs& a, cudaStream_t stream);
cudaError_t launch_attn_f32(const AttnArgs& a, bool prefix, cudaStream_t stream);
// How the tile kernel divides its work: query tiles per block (two, unless blocks of one
// still fit the SMs), splits of the slots, and whether a block of one tile takes its
// steps in two interleaved halves.
struct TileSplit {
  int tiles, splits;
  bool paired;
};
cudaError_t launch_attn_status(const AttnArgs& a, cudaStream_t stream);
cudaError_t launch_attn_tile(const AttnArgs& a, bool prefix, const TileSplit& split, cudaStream_t stream);
cudaError_t launch_attn_token(const AttnArgs& a, int blocks, cudaStream_t stream);
// How the kernel over 4-bit records takes a head's query rows: column tiles of eight per warp, groups of
// so many rows as units of their own; and whether tiles of 16 slots (not 32) let every chunk have its own block.
struct RecordRows {
  int tiles, groups;
  bool fits;
};
cudaError_t launch_attn_record(const AttnArgs& a, const RecordRows& rows, cudaStream_t stream);
cudaError_t launch_weights16(const AttnArgs& a, cudaStream_t stream);
cudaError_t launch_scores_weights(const AttnArgs& a, cudaStream_t stream);
cudaError_t launch_attn_combine(const AttnArgs& a, cudaStream_t stream);
cudaError_t launch_attn_weights(const AttnArgs& a, cudaStream_t stream);

}  // namespace sv
