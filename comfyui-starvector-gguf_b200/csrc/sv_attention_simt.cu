// sv_attention_simt.cu -- attention over the cache on the FP32 pipes.
//
// o = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m), s_j = (q . k_j) * scale * log2 e, in
// one pass over the slots with the running maximum m and sum.  A block of 256 threads
// holds BM query rows (16 or 64, of one key/value head's group) and walks 64-slot
// tiles staged in shared memory as float; a thread owns BM / 16 rows by 4 slots of
// the scores and BM / 16 rows by 8 dimensions of the output.
#include "sv_attention.h"

namespace sv {
namespace {

constexpr int NT = 256;
constexpr int BN = 64;                  // slots per tile
constexpr int KS = kAttnMaxDim + 4;     // row stride of the staged queries and keys (floats)
constexpr int VS = kAttnMaxDim;
constexpr int PS = BN + 4;

template <int BM> constexpr size_t simt_smem() { return sizeof(float) * (BM * KS + BN * KS + BN * VS + BM * PS); }

// Stages `count` rows of `dim` elements as float, zeros past `valid` rows.
template <typename T>
__device__ __forceinline__ void stage(float* dst, int stride, const T* src, int64_t src_stride, int count, int valid,
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

template <typename T>
__device__ __forceinline__ const T* query_row(const AttnArgs& a, int r, int h, int m) {
  const int i = m / a.group, g = m - i * a.group;
  return static_cast<const T*>(a.q) + r * a.q_row + i * a.q_tok + (int64_t)(h * a.group + g) * a.q_head;
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

template <typename T, int BM>
__global__ void __launch_bounds__(NT) attn_simt_kernel(const AttnArgs a, const bool prefix) {
  constexpr int RPT = BM / 16;
  extern __shared__ float4 smem4[];
  float* qs = reinterpret_cast<float*>(smem4);
  float* ks = qs + BM * KS;
  float* vs = ks + BN * KS;
  float* ps = vs + BN * VS;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int nG = a.n * a.group;
  const int rows_m = prefix ? a.rows * nG : nG;  // query rows of this unit
  const int S = prefix ? a.p_splits : max(a.o_splits, 1);
  const int split = blockIdx.x % S, m0 = (blockIdx.x / S) * BM;
  const int unit = blockIdx.y;
  const int h = prefix ? unit : unit % a.kv_heads, r_own = prefix ? 0 : unit / a.kv_heads;
  const int mlast = min(m0 + BM, rows_m) - 1;

  // Queries, each scaled by nothing: the scale is applied to the f32 score.
  {
    const int vec = a.dim >> 3;
    for (int x = threadIdx.x; x < BM * vec; x += NT) {
      const int row = x / vec, c = (x - row * vec) * 8, m = m0 + row;
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (m < rows_m) load8(query_row<T>(a, prefix ? m / nG : r_own, h, prefix ? m % nG : m) + c, f);
      float4* d = reinterpret_cast<float4*>(qs + row * KS + c);
      d[0] = make_float4(f[0], f[1], f[2], f[3]);
      d[1] = make_float4(f[4], f[5], f[6], f[7]);
    }
  }

  // The slots: [a0, a1) are sinks before the window, [b0, b1) the rest.
  RowSpan sp = {0, a.prefix};
  int a0 = 0, a1 = 0, b0 = 0, b1 = a.prefix;
  if (!prefix) {
    sp = row_span(a, r_own);
    const int pf = sp.end - a.n + m0 / a.group, pl = sp.end - a.n + mlast / a.group;
    b0 = window_low(a, sp.start, pf);
    b1 = max(pl + 1, b0);
    a0 = sp.start;
    a1 = pl >= sp.start ? max(a0, min(sp.start + a.sinks, b0)) : a0;
    if (pl < sp.start) b1 = b0;
  }
  const int ta = (a1 - a0 + BN - 1) / BN, tiles = ta + (b1 - b0 + BN - 1) / BN;
  const int t0 = (int)((int64_t)tiles * split / S), t1 = (int)((int64_t)tiles * (split + 1) / S);
  const T* kb = static_cast<const T*>(prefix ? a.pk : a.k);
  const T* vb = static_cast<const T*>(prefix ? a.pv : a.v);
  const int64_t slot = prefix ? a.p_slot : a.kv_slot;
  const int64_t base = prefix ? h * a.p_head : r_own * a.kv_row + h * a.kv_head;

  float m[RPT], l[RPT], o[RPT][8];
  int pos[RPT], low[RPT];
#pragma unroll
  for (int r = 0; r < RPT; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int c = 0; c < 8; ++c) o[r][c] = 0.f;
    pos[r] = prefix ? a.prefix : sp.end - a.n + (m0 + ty * RPT + r) / a.group;
    low[r] = prefix ? 0 : window_low(a, sp.start, pos[r]);
  }
  for (int t = t0; t < t1; ++t) {
    const bool in_a = t < ta;
    const int j0 = in_a ? a0 + t * BN : b0 + (t - ta) * BN;
    const int valid = min(BN, (in_a ? a1 : b1) - j0);
    __syncthreads();
    stage(ks, KS, kb + base + j0 * slot, slot, BN, valid, a.dim);
    stage(vs, VS, vb + base + j0 * slot, slot, BN, valid, a.dim);
    __syncthreads();
    float s[RPT][4];
    scores<RPT>(qs, ks, ty, tx, a.dim, s);
#pragma unroll
    for (int r = 0; r < RPT; ++r) {
      float mx = m[r];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int j = j0 + tx + 16 * c;
        const bool see = tx + 16 * c < valid && (prefix || slot_seen(a, sp.start, pos[r], low[r], j));
        s[r][c] = see ? s[r][c] * a.scale : -INFINITY;
        mx = fmaxf(mx, s[r][c]);
      }
#pragma unroll
      for (int k = 1; k < 16; k <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
      const float ref = mx == -INFINITY ? 0.f : mx;  // nothing seen yet: every weight is zero
      const float f = exp2f(m[r] - ref);
      m[r] = mx;
      l[r] *= f;
#pragma unroll
      for (int c = 0; c < 8; ++c) o[r][c] *= f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float p = exp2f(s[r][c] - ref);
        l[r] += p;
        ps[(ty * RPT + r) * PS + tx + 16 * c] = p;
      }
    }
    __syncwarp();  // a warp's rows of ps are read by that warp alone
    for (int j = 0; j < valid; ++j) {
      const float4 v0 = *reinterpret_cast<const float4*>(vs + j * VS + tx * 4);
      const float4 v1 = *reinterpret_cast<const float4*>(vs + j * VS + 64 + tx * 4);
#pragma unroll
      for (int r = 0; r < RPT; ++r) {
        const float p = ps[(ty * RPT + r) * PS + j];
        if (p != 0.f) {  // what is hidden adds nothing, whatever its slot holds
          o[r][0] = fmaf(p, v0.x, o[r][0]);
          o[r][1] = fmaf(p, v0.y, o[r][1]);
          o[r][2] = fmaf(p, v0.z, o[r][2]);
          o[r][3] = fmaf(p, v0.w, o[r][3]);
          o[r][4] = fmaf(p, v1.x, o[r][4]);
          o[r][5] = fmaf(p, v1.y, o[r][5]);
          o[r][6] = fmaf(p, v1.z, o[r][6]);
          o[r][7] = fmaf(p, v1.w, o[r][7]);
        }
      }
    }
    __syncwarp();
  }
  const bool direct = !prefix && a.o_splits == 0;
  const int64_t all = (int64_t)a.rows * a.kv_heads * nG;
#pragma unroll
  for (int r = 0; r < RPT; ++r) {
#pragma unroll
    for (int k = 1; k < 16; k <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], k);
    const int mm = m0 + ty * RPT + r;
    if (mm >= rows_m) continue;
    const int row = prefix ? mm / nG : r_own, mr = prefix ? mm % nG : mm;
    const int64_t idx = ((int64_t)row * a.kv_heads + h) * nG + mr;
    if (direct) {
      const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
      const int i = mr / a.group, g = mr - i * a.group;
      T* out = static_cast<T*>(a.out) + (((int64_t)row * a.n + i) * a.heads + h * a.group + g) * a.dim;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const int d = (c >> 2) * 64 + tx * 4 + (c & 3);
        if (d < a.dim) out[d] = from_float<T>(o[r][c] * inv);
      }
      if (a.lse && tx == 0) a.lse[idx] = l[r] == 0.f ? INFINITY : m[r] + log2f(l[r]);
    } else {
      const int64_t at = (int64_t)split * all + (prefix ? prefix_index(a, row, h, mr) : idx);
      float* out = (prefix ? a.prefix_o : a.part_o) + at * a.dim;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const int d = (c >> 2) * 64 + tx * 4 + (c & 3);
        if (d < a.dim) out[d] = o[r][c];
      }
      if (tx == 0) (prefix ? a.prefix_ml : a.part_ml)[at] = make_float2(m[r], l[r]);
    }
  }
  if (a.status && !prefix && threadIdx.x == 0 && blockIdx.x == 0 && h == 0) {
    const int e = a.lengths ? a.lengths[r_own] : a.capacity, s = a.starts ? a.starts[r_own] : 0;
    a.status[r_own] = (e < 0 || e > a.capacity || s < 0 || s > max(e, 0)) ? 8 : 0;
  }
}

// Accumulated weights: w[slot] += sum over the group's rows of 2^(s - lse).  One block
// owns 64 slots of one row and head and walks the query rows, so the sum's order is
// fixed and no atomics are needed.
template <typename T>
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
  const int64_t base = r * a.kv_row + h * a.kv_head + j0 * a.kv_slot;
  stage(ks, KS, static_cast<const T*>(a.k) + base, a.kv_slot, BN, valid, a.dim);
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  for (int m0 = 0; m0 < nG; m0 += BM) {
    __syncthreads();
    const int vec = a.dim >> 3;
    for (int x = threadIdx.x; x < BM * vec; x += NT) {
      const int row = x / vec, c = (x - row * vec) * 8;
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (m0 + row < nG) load8(query_row<T>(a, r, h, m0 + row) + c, f);
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
      if (m >= nG) continue;
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
    a.weights[r * a.w_row + h * a.w_head + j0 + threadIdx.x] += t;
  }
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

template <typename T, int BM> cudaError_t simt(const AttnArgs& a, bool prefix, cudaStream_t stream) {
  const int64_t rows_m = (int64_t)(prefix ? a.rows : 1) * a.n * a.group;
  const int64_t S = prefix ? a.p_splits : (a.o_splits ? a.o_splits : 1);
  const dim3 grid((unsigned)((rows_m + BM - 1) / BM * S), (unsigned)(prefix ? a.kv_heads : a.rows * a.kv_heads));
  constexpr size_t smem = simt_smem<BM>();
  cudaError_t e = allow_smem<attn_simt_kernel<T, BM>>(smem);
  if (e != cudaSuccess) return e;
  attn_simt_kernel<T, BM><<<grid, NT, smem, stream>>>(a, prefix);
  return cudaGetLastError();
}

template <typename T> cudaError_t simt_any(const AttnArgs& a, bool prefix, cudaStream_t stream) {
  const int64_t rows_m = (int64_t)(prefix ? a.rows : 1) * a.n * a.group;
  return rows_m <= 16 ? simt<T, 16>(a, prefix, stream) : simt<T, 64>(a, prefix, stream);
}

template <typename T> cudaError_t weights_any(const AttnArgs& a, cudaStream_t stream) {
  constexpr size_t smem = sizeof(float) * (64 * KS + BN * KS + 16 * BN);
  cudaError_t e = allow_smem<attn_weights_kernel<T>>(smem);
  if (e != cudaSuccess) return e;
  const dim3 grid((unsigned)((a.capacity + BN - 1) / BN), (unsigned)(a.rows * a.kv_heads));
  attn_weights_kernel<T><<<grid, NT, smem, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_attn_simt(const AttnArgs& a, bool prefix, cudaStream_t stream) {
  return simt_any<float>(a, prefix, stream);
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

cudaError_t launch_attn_weights(const AttnArgs& a, cudaStream_t stream) {
  switch (a.dtype) {
    case 0: return weights_any<float>(a, stream);
    case 1: return weights_any<__half>(a, stream);
    default: return weights_any<__nv_bfloat16>(a, stream);
  }
}

}  // namespace sv
