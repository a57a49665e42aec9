// sv_attention_join.cu -- what follows the attention kernels: the join of parts that
// were split over the slots, and the accumulated weights of calls with many queries.
#include "../../include/starvector_sampling.h"
#include "sv_attention.h"

namespace sv {
namespace {

constexpr int NT = 256;
constexpr int BN = 64;                  // slots per tile
constexpr int KS = kAttnMaxDim + 4;     // row stride of the staged queries and keys (floats)

// Stages `count` rows of `dim` elements as float, zeros past `valid` rows.
__device__ __forceinline__ void stage(float* dst, int stride, const float* src, int64_t src_stride, int count, int valid,
                                      int dim) {
  const int vec = dim >> 3;
  for (int x = threadIdx.x; x < count * vec; x += NT) {
    const int row = x / vec, c = (x - row * vec) * 8;
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (row < valid) load8(src + row * src_stride + c, f);
    float4* d = reinterpret_cast<float4*>(dst + row * stride + c);
    d[0] = make_float4(f[0], f[1], f[2], f[3]);
    d[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
}

__device__ __forceinline__ const float* query_row(const AttnArgs& a, int r, int h, int m) {
  const int i = m / a.group, g = m - i * a.group;
  return static_cast<const float*>(a.q) + r * a.q_row + i * a.q_tok + (int64_t)(h * a.group + g) * a.q_head;
}

// Scores of RPT rows x 4 slots (slots tx, tx + 16, ...) of the staged tiles.
template <int RPT>
__device__ __forceinline__ void scores(const float* qs, const float* ks, int ty, int tx, int dim, float (&s)[RPT][4]) {
#pragma unroll
  for (int r = 0; r < RPT; ++r)
#pragma unroll
    for (int c = 0; c < 4; ++c) s[r][c] = 0.f;
  for (int d = 0; d < dim; d += 4) {
    float4 q[RPT], k[4];
#pragma unroll
    for (int r = 0; r < RPT; ++r) q[r] = *reinterpret_cast<const float4*>(qs + (ty * RPT + r) * KS + d);
#pragma unroll
    for (int c = 0; c < 4; ++c) k[c] = *reinterpret_cast<const float4*>(ks + (tx + 16 * c) * KS + d);
#pragma unroll
    for (int r = 0; r < RPT; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        s[r][c] = fmaf(q[r].x, k[c].x, fmaf(q[r].y, k[c].y, fmaf(q[r].z, k[c].z, fmaf(q[r].w, k[c].w, s[r][c]))));
  }
}

// Accumulated weights of float calls, on the FP32 pipes: w[slot] += sum over the group's
// rows of 2^(s - lse).  One block owns 64 slots of one row and head and walks (a split
// of) the query rows, so the sum's order is fixed and no atomics are needed.
__global__ void __launch_bounds__(NT) attn_weights_kernel(const AttnArgs a) {
  constexpr int BM = 64, RPT = BM / 16;
  extern __shared__ float4 smem4[];
  float* qs = reinterpret_cast<float*>(smem4);
  float* ks = qs + BM * KS;
  float* sums = ks + BN * KS;  // [16][BN]
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int nG = a.n * a.group;
  const int unit = blockIdx.y, h = unit % a.kv_heads, r = unit / a.kv_heads;
  const RowSpan sp = row_span(a, r);
  const int j0 = blockIdx.x * BN;
  const int valid = min(BN, sp.end - j0);
  if (valid <= 0) return;
  int m_first, m_end;
  weight_rows(a, sp, j0, valid, blockIdx.z, m_first, m_end);
  const int64_t base = r * a.kv_row + h * a.kv_head + j0 * a.kv_slot;
  stage(ks, KS, static_cast<const float*>(a.k) + base, a.kv_slot, BN, valid, a.dim);
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  for (int m0 = m_first; m0 < m_end; m0 += BM) {
    __syncthreads();
    const int vec = a.dim >> 3;
    for (int x = threadIdx.x; x < BM * vec; x += NT) {
      const int row = x / vec, c = (x - row * vec) * 8;
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (m0 + row < m_end) load8(query_row(a, r, h, m0 + row) + c, f);
      float4* d = reinterpret_cast<float4*>(qs + row * KS + c);
      d[0] = make_float4(f[0], f[1], f[2], f[3]);
      d[1] = make_float4(f[4], f[5], f[6], f[7]);
    }
    __syncthreads();
    float s[RPT][4];
    scores<RPT>(qs, ks, ty, tx, a.dim, s);
#pragma unroll
    for (int k = 0; k < RPT; ++k) {
      const int m = m0 + ty * RPT + k;
      if (m >= m_end) continue;
      const int p = sp.end - a.n + m / a.group, lo = window_low(a, sp.start, p);
      const float lse = a.lse[(int64_t)unit * nG + m];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (slot_seen(a, sp.start, p, lo, j0 + tx + 16 * c)) sum[c] += exp2f(s[k][c] * a.scale - lse);
    }
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) sums[ty * BN + tx + 16 * c] = sum[c];
  __syncthreads();
  if (threadIdx.x < valid) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) t += sums[k * BN + threadIdx.x];
    if (j0 + (int)threadIdx.x >= sp.start) add_weight(a, unit, r, h, j0 + threadIdx.x, blockIdx.z, t);
  }
}

// The splits of the weights' sums, in order: one thread per slot.
__global__ void __launch_bounds__(NT) weights_sum_kernel(const AttnArgs a) {
  const int unit = blockIdx.y, h = unit % a.kv_heads, r = unit / a.kv_heads;
  const RowSpan sp = row_span(a, r);
  const int j = blockIdx.x * NT + threadIdx.x;
  if (j < sp.start || j >= sp.end) return;
  float t = 0.f;
#pragma unroll 8
  for (int s = 0; s < a.w_splits; ++s)
    t += a.weight_parts[((int64_t)s * a.rows * a.kv_heads + unit) * a.capacity + j];
  a.weights[r * a.w_row + h * a.w_head + j] += t;
}

// The rows' statuses ahead of the tile kernel, any of whose blocks may then report that it gave up.
__global__ void __launch_bounds__(NT) attn_status_kernel(const AttnArgs a) {
  const int r = blockIdx.x * NT + threadIdx.x;
  if (r >= a.rows) return;
  const int e = a.lengths ? a.lengths[r] : a.capacity, s = a.starts ? a.starts[r] : 0;
  a.status[r] = (e < 0 || e > a.capacity || s < 0 || s > max(e, 0)) ? SV_ST_LENGTH : 0;
}

// Joins the splits of one query row per warp: a lane holds four dimensions.
template <typename T>
__global__ void __launch_bounds__(NT) attn_combine_kernel(const AttnArgs a) {
  const int nG = a.n * a.group, S = a.p_splits + a.o_splits;
  const int64_t all = (int64_t)a.rows * a.kv_heads * nG;
  const int64_t idx = (int64_t)blockIdx.x * (NT / 32) + (threadIdx.x >> 5);
  if (idx >= all) return;
  const int lane = threadIdx.x & 31, d = lane * 4;
  float mx = -INFINITY;
  const int64_t unit = idx / nG;
  const int m = (int)(idx - unit * nG), i = m / a.group, g = m - i * a.group;
  const int h = (int)(unit % a.kv_heads), r = (int)(unit / a.kv_heads);
  const int64_t pidx = prefix_index(a, r, h, m);
  auto ml_of = [&](int s) {
    return s < a.p_splits ? a.prefix_ml[s * all + pidx] : a.part_ml[(s - a.p_splits) * all + idx];
  };
  for (int s = lane; s < S; s += 32) mx = fmaxf(mx, ml_of(s).x);
#pragma unroll
  for (int k = 1; k < 32; k <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
  const float ref = mx == -INFINITY ? 0.f : mx;
  float l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < S; ++s) {
    const float2 ml = ml_of(s);
    if (ml.y == 0.f) continue;  // the split saw nothing
    const float f = exp2f(ml.x - ref);
    l = fmaf(ml.y, f, l);
    if (d < a.dim) {
      const float* part = s < a.p_splits ? a.prefix_o + (s * all + pidx) * a.dim
                                         : a.part_o + ((s - a.p_splits) * all + idx) * a.dim;
      const float4 x = *reinterpret_cast<const float4*>(part + d);
      o.x = fmaf(x.x, f, o.x);
      o.y = fmaf(x.y, f, o.y);
      o.z = fmaf(x.z, f, o.z);
      o.w = fmaf(x.w, f, o.w);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (d < a.dim) {
    T* out = static_cast<T*>(a.out) + (((int64_t)r * a.n + i) * a.heads + h * a.group + g) * a.dim + d;
    out[0] = from_float<T>(o.x * inv);
    out[1] = from_float<T>(o.y * inv);
    out[2] = from_float<T>(o.z * inv);
    out[3] = from_float<T>(o.w * inv);
  }
  if (a.lse && lane == 0) a.lse[idx] = l == 0.f ? INFINITY : mx + log2f(l);
}

}  // namespace

cudaError_t launch_attn_status(const AttnArgs& a, cudaStream_t stream) {
  attn_status_kernel<<<(unsigned)((a.rows + NT - 1) / NT), NT, 0, stream>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_attn_combine(const AttnArgs& a, cudaStream_t stream) {
  const int64_t all = (int64_t)a.rows * a.n * a.heads;
  const unsigned grid = (unsigned)((all + NT / 32 - 1) / (NT / 32));
  switch (a.dtype) {
    case 0: attn_combine_kernel<float><<<grid, NT, 0, stream>>>(a); break;
    case 1: attn_combine_kernel<__half><<<grid, NT, 0, stream>>>(a); break;
    default: attn_combine_kernel<__nv_bfloat16><<<grid, NT, 0, stream>>>(a); break;
  }
  return cudaGetLastError();
}

cudaError_t launch_weights_sum(const AttnArgs& a, cudaStream_t stream) {
  weights_sum_kernel<<<dim3((unsigned)((a.capacity + NT - 1) / NT), (unsigned)(a.rows * a.kv_heads)), NT, 0, stream>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_attn_weights(const AttnArgs& a, cudaStream_t stream) {
  constexpr size_t smem = sizeof(float) * (64 * KS + BN * KS + 16 * BN);
  const cudaError_t e = allow_smem<attn_weights_kernel>(smem);
  if (e != cudaSuccess) return e;
  const dim3 grid((unsigned)((a.capacity + BN - 1) / BN), (unsigned)(a.rows * a.kv_heads), (unsigned)a.w_splits);
  attn_weights_kernel<<<grid, NT, smem, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace sv
