// sv_attention_f32.cu -- attention over the cache for float queries and caches, at any
// number of query rows, on the tensor cores with split operands.
//
// Mathematics: one pass with a running reference, as the 16-bit kernels (o = sum_j
// 2^(s_j - ref) v_j, l = sum_j 2^(s_j - ref); ref follows the maximum once a score
// exceeds it by 2^8).  Every f32 operand x is taken as hi + lo, hi x rounded to 11
// significant bits and lo = x - hi (exact; the tensor core reads its upper 11 bits):
// x y = hi hi + hi lo + lo hi with a relative error of about 2^-22 per product, sums in
// f32; three products m16n8k8 (TF32) per step.  Rounded halves and scores summed outside the
// tensor core take 98 us for 2 x 333 queries over 512 slots, truncated ones 94 us with more
// error (1.6e-6 of the output for 24 rows over 1460 shared slots, and 3.2e-7 rounded).  On the
// FP32 pipes the same work took 140 us.  An operand that is not finite (or, a key, that
// rounds to infinity) has no such split: it is computed value by value instead.  (A query that is not finite makes its row NaN, as an infinite score does.)
//
// A block of 8 warps holds 16 query rows of one key/value head's group and takes the
// slots 8 per warp and round, straight from global memory into the fragments (as in the
// token kernel: the sum over dimensions in any order, output columns in any order);
// the queries' halves are in shared memory in the fragments' order.  What bounds it: the
// products (192 per 16 slots and warp) for prompts, the cache's bytes for single tokens.
#include "sv_attention.h"

namespace sv {
namespace {

constexpr int NW = 8, NT = NW * 32;
constexpr int BM = 16, TK = 8;
constexpr float kSlack = 8.f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma(float (&c)[4], float a0, float a1, float a2, float a3, float b0, float b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
               "{%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(__float_as_uint(a0)), "r"(__float_as_uint(a1)), "r"(__float_as_uint(a2)),
                 "r"(__float_as_uint(a3)), "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}

// Truncated, not rounded: the type's largest values must not become infinite.
__device__ __forceinline__ float upper(float x) { return __uint_as_float(__float_as_uint(x) & 0xffffe000u); }
// Rounded (ties away), for queries, keys and weights: their lower halves then have either
// sign, where truncated ones have their number's, and the dropped lo lo and the lower halves'
// own truncation would make every score too small by some 2^-22 of itself.  Below kRoundable only.
constexpr float kRoundable = 0x1.ffep127f;
__device__ __forceinline__ float nearest(float x) { return __uint_as_float((__float_as_uint(x) + 0x1000u) & 0xffffe000u); }
__device__ __forceinline__ float4 nearest(float4 x) {
  return make_float4(nearest(x.x), nearest(x.y), nearest(x.z), nearest(x.w));
}
__device__ __forceinline__ float4 upper(float4 x) { return make_float4(upper(x.x), upper(x.y), upper(x.z), upper(x.w)); }
__device__ __forceinline__ float4 minus(float4 a, float4 b) {
  return make_float4(a.x - b.x, a.y - b.y, a.z - b.z, a.w - b.w);
}
__device__ __forceinline__ float4 load_stream(const float* p, bool ok) {
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (ok)
    asm volatile("ld.global.nc.L1::no_allocate.v4.f32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "l"(p));
  return v;
}
__device__ __forceinline__ float finite(float x) { return fabsf(x) < INFINITY ? x : 0.f; }
__device__ __forceinline__ float roundable(float x) { return fabsf(x) < kRoundable ? x : 0.f; }
__device__ __forceinline__ float4 roundable(float4 x) {
  return make_float4(roundable(x.x), roundable(x.y), roundable(x.z), roundable(x.w));
}
__device__ __forceinline__ float4 finite(float4 x) { return make_float4(finite(x.x), finite(x.y), finite(x.z), finite(x.w)); }
// The largest magnitude of four values and m, NaN if one is NaN.
__device__ __forceinline__ float widest(float4 v, float m) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(v.x)), "f"(m));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(v.y)), "f"(r));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(v.z)), "f"(r));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(v.w)), "f"(r));
  return r;
}

template <int DC, bool FULL>
__global__ void __launch_bounds__(NT, 1) attn_f32_kernel(const __grid_constant__ AttnArgs a, const bool prefix) {
  constexpr int KU = 4 * DC, VU = 2 * DC, OS = 64 * DC;  // vectors of 4 dimensions: per key, per value; output row
  extern __shared__ float4 dyn[];                        // queries [hi, lo][KU][2][32], later the warps' outputs
  __shared__ float2 warp_ml[NW][BM];
  __shared__ float factor[NW][BM];
  __shared__ float2 joined[BM];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int nG = a.n * a.group, D = a.dim;
  const int rows_m = prefix ? a.rows * nG : nG;
  const int S = prefix ? a.p_splits : max(a.o_splits, 1);
  // The last rows see the most slots under a causal mask: they start first.
  const int split = blockIdx.x % S, m0 = (gridDim.x / S - 1 - blockIdx.x / S) * BM;
  const int unit = blockIdx.y;
  const int h = prefix ? unit : unit % a.kv_heads, r_own = prefix ? 0 : unit / a.kv_heads;

  auto query = [&](int m) {
    const int r = prefix ? m / nG : r_own, mr = prefix ? m - r * nG : m, i = mr / a.group;
    return static_cast<const float*>(a.q) + r * a.q_row + i * a.q_tok + (int64_t)(h * a.group + mr - i * a.group) * a.q_head;
  };
  for (int x = tid; x < KU * 64; x += NT) {
    const int ln = x & 31, y = (x >> 5) & 1, u = x >> 6, m = m0 + (ln >> 2) + 8 * y, d = 16 * u + 4 * (ln & 3);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (m < rows_m && (FULL || d < D)) v = __ldg(reinterpret_cast<const float4*>(query(m) + d));
    auto half = [](float x) { return fabsf(x) < kRoundable ? nearest(x) : upper(x); };
    const float4 hi = make_float4(half(v.x), half(v.y), half(v.z), half(v.w));
    dyn[(u * 2 + y) * 32 + ln] = hi;
    dyn[((KU + u) * 2 + y) * 32 + ln] = minus(v, hi);
  }
  __syncthreads();

  // The slots: [a0, a1) are sinks before the window, [b0, b1) the rest.
  const int m_last = min(m0 + BM, rows_m) - 1;
  RowSpan sp = {0, a.prefix};
  int a0 = 0, a1 = 0, b0 = 0, b1 = a.prefix, pos_first = 0, low_last = 0;
  if (!prefix) {
    sp = row_span(a, r_own);
    const int pl = sp.end - a.n + m_last / a.group;
    pos_first = sp.end - a.n + m0 / a.group;
    b0 = window_low(a, sp.start, pos_first);
    b1 = pl < sp.start ? b0 : max(pl + 1, b0);
    a0 = sp.start;
    a1 = pl >= sp.start ? max(a0, min(sp.start + a.sinks, b0)) : a0;
    low_last = window_low(a, sp.start, pl);
  }
  const int ta = (a1 - a0 + TK - 1) / TK, tiles = ta + (b1 - b0 + TK - 1) / TK;
  const int t0 = (int)((int64_t)tiles * split / S), t1 = (int)((int64_t)tiles * (split + 1) / S);
  const int64_t slot = prefix ? a.p_slot : a.kv_slot, base = prefix ? h * a.p_head : r_own * a.kv_row + h * a.kv_head;
  const float* kb = static_cast<const float*>(prefix ? a.pk : a.k) + base;
  const float* vb = static_cast<const float*>(prefix ? a.pv : a.v) + base;
  int pos[2], low[2];
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    pos[y] = prefix ? a.prefix : sp.end - a.n + (m0 + g + 8 * y) / a.group;
    low[y] = prefix ? 0 : window_low(a, sp.start, pos[y]);
  }
  auto tile_at = [&](int tile, int& j0, int& jend) {
    const bool in_a = tile < ta;
    j0 = in_a ? a0 + tile * TK : b0 + (tile - ta) * TK;
    jend = in_a ? a1 : b1;
  };
  float4 kf[KU], vf[2][VU];
  auto load_k = [&](int tile) {
    int j0, jend;
    tile_at(tile, j0, jend);
    const int j = j0 + g;
    const float* src = kb + j * slot + 4 * t;
#pragma unroll
    for (int u = 0; u < KU; ++u) kf[u] = load_stream(src + 16 * u, tile < t1 && j < jend && (FULL || 16 * u + 4 * t < D));
  };
  auto load_v = [&](int tile) {
    int j0, jend;
    tile_at(tile, j0, jend);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int j = j0 + 2 * t + x;
      const float* src = vb + j * slot + 4 * g;
#pragma unroll
      for (int u = 0; u < VU; ++u)
        vf[x][u] = load_stream(src + 32 * u, tile < t1 && j < jend && (FULL || 32 * u + 4 * g < D));
    }
  };

  float o[4 * VU][4];
#pragma unroll
  for (int j = 0; j < 4 * VU; ++j)
#pragma unroll
    for (int x = 0; x < 4; ++x) o[j][x] = 0.f;
  float ref[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  load_k(t0 + warp);
  load_v(t0 + warp);
  for (int tile = t0 + warp; tile < t1; tile += NW) {
    int j0, jend;
    tile_at(tile, j0, jend);
    float wide = 0.f;
#pragma unroll
    for (int u = 0; u < KU; ++u) wide = widest(kf[u], wide);
    const unsigned bad_k = __ballot_sync(0xffffffffu, !(wide < kRoundable));
    if (bad_k) {
#pragma unroll
      for (int u = 0; u < KU; ++u) kf[u] = roundable(kf[u]);
    }
    float s[4];
    {
      // Sums of their own for the halves' products (a product waits for the one before it in
      // the same sum); those of the upper halves are added in f32 with rounding, as the
      // tensor core truncates as it adds.
      float c[2][4], e[2][4];
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int k = 0; k < 4; ++k) c[x][k] = e[x][k] = 0.f;
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        const float4 qh0 = dyn[u * 64 + lane], qh1 = dyn[u * 64 + 32 + lane];
        const float4 ql0 = dyn[(KU + u) * 64 + lane], ql1 = dyn[(KU + u) * 64 + 32 + lane];
        const float4 kh = nearest(kf[u]), kl = minus(kf[u], kh);
        float d[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        mma(d[0], qh0.x, qh1.x, qh0.y, qh1.y, kh.x, kh.y);
        mma(d[1], qh0.z, qh1.z, qh0.w, qh1.w, kh.z, kh.w);
        mma(c[0], qh0.x, qh1.x, qh0.y, qh1.y, kl.x, kl.y);
        mma(c[1], ql0.x, ql1.x, ql0.y, ql1.y, kh.x, kh.y);
        mma(c[0], qh0.z, qh1.z, qh0.w, qh1.w, kl.z, kl.w);
        mma(c[1], ql0.z, ql1.z, ql0.w, ql1.w, kh.z, kh.w);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          e[0][k] += d[0][k];
          e[1][k] += d[1][k];
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) s[k] = (e[0][k] + e[1][k]) + (c[0][k] + c[1][k]);
    }
    if (bad_k) {  // the slots whose keys are not finite, value by value
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int e = 2 * t + (k & 1), j = j0 + e, m = m0 + g + 8 * (k >> 1);
        if (!(bad_k >> (4 * e) & 15u) || m >= rows_m) continue;
        float x = 0.f;
        for (int d = 0; d < D; ++d) x = fmaf(__ldg(query(m) + d), __ldg(kb + j * slot + d), x);
        s[k] = x;
      }
      __syncwarp();
    }
    load_k(tile + NW);
    const bool whole = j0 + TK <= jend && (prefix || tile < ta || (j0 >= low_last && j0 + TK - 1 <= pos_first));
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      s[k] *= a.scale;
      if (!whole) {
        const int j = j0 + 2 * t + (k & 1);
        if (j >= jend || (!prefix && !slot_seen(a, sp.start, pos[k >> 1], low[k >> 1], j))) s[k] = -INFINITY;
      }
    }
    float mx[2] = {fmaxf(s[0], s[1]), fmaxf(s[2], s[3])};
    if (__any_sync(0xffffffffu, mx[0] > ref[0] + kSlack || mx[1] > ref[1] + kSlack)) {
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        mx[y] = fmaxf(mx[y], __shfl_xor_sync(0xffffffffu, mx[y], 1));
        mx[y] = fmaxf(mx[y], __shfl_xor_sync(0xffffffffu, mx[y], 2));
        const float now = fmaxf(mx[y], ref[y]);
        const float f = now == ref[y] ? 1.f : ex2(ref[y] - now);
        ref[y] = now;
        l[y] *= f;
#pragma unroll
        for (int j = 0; j < 4 * VU; ++j) {
          o[j][2 * y] *= f;
          o[j][2 * y + 1] *= f;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float at = ref[k >> 1] == -INFINITY ? 0.f : ref[k >> 1];
      s[k] = ex2(s[k] - at);
      l[k >> 1] += s[k];
    }
    wide = 0.f;
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int u = 0; u < VU; ++u) wide = widest(vf[x][u], wide);
    if (__any_sync(0xffffffffu, !(wide < INFINITY))) {
      // A value is not finite: the product takes a zero in its place (or it would reach rows
      // that do not see it), and the rows that see it get it here.
#pragma unroll 1
      for (int e = 0; e < TK; ++e) {
        const int from = (lane & 28) | (e >> 1), j = j0 + e;
        float w[2];
        bool sees[2];  // (a weight may be zero)
#pragma unroll
        for (int y = 0; y < 2; ++y) sees[y] = prefix || slot_seen(a, sp.start, pos[y], low[y], j);
#pragma unroll
        for (int y = 0; y < 2; ++y) w[y] = __shfl_sync(0xffffffffu, e & 1 ? s[2 * y + 1] : s[2 * y], from);
        if (j >= jend) break;
#pragma unroll
        for (int u = 0; u < VU; ++u)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int d = 32 * u + 8 * t + 4 * x;
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            if (FULL || d < D) {
              const float4 f = __ldg(reinterpret_cast<const float4*>(vb + j * slot + d));
              v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int y = 0; y < 2; ++y)
                if (sees[y] && !isfinite(v[k])) o[4 * u + k][2 * y + x] = fmaf(w[y], v[k], o[4 * u + k][2 * y + x]);
          }
      }
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int u = 0; u < VU; ++u) vf[x][u] = finite(vf[x][u]);
    }
    // Weights as the A operand: slot 2 t is its column t, slot 2 t + 1 its column t + 4.
    float ph[4], pl[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      ph[k] = nearest(s[k]);
      pl[k] = s[k] - ph[k];
    }
#pragma unroll
    for (int u = 0; u < VU; ++u) {
      const float4 h0 = upper(vf[0][u]), h1 = upper(vf[1][u]), l0 = minus(vf[0][u], h0), l1 = minus(vf[1][u], h1);
      // A tile's products in a sum of their own, added in f32 with rounding: the tensor core
      // truncates as it adds, which over many slots would pull the output towards zero.
#define SV_PV(e, f)                                     \
  {                                                     \
    float c[4] = {0.f, 0.f, 0.f, 0.f};                  \
    mma(c, pl[0], pl[2], pl[1], pl[3], h0.f, h1.f);     \
    mma(c, ph[0], ph[2], ph[1], ph[3], l0.f, l1.f);     \
    mma(c, ph[0], ph[2], ph[1], ph[3], h0.f, h1.f);     \
    for (int k = 0; k < 4; ++k) o[4 * u + e][k] += c[k]; \
  }
      SV_PV(0, x) SV_PV(1, y) SV_PV(2, z) SV_PV(3, w)
#undef SV_PV
    }
    load_v(tile + NW);
  }

  // The warps' results, joined through shared memory: a thread holds 8 consecutive
  // dimensions of each 32 for its two rows.
  __syncthreads();
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    l[y] += __shfl_xor_sync(0xffffffffu, l[y], 1);
    l[y] += __shfl_xor_sync(0xffffffffu, l[y], 2);
    const int m = g + 8 * y;
    if (t == 0) warp_ml[warp][m] = make_float2(ref[y], l[y]);
#pragma unroll
    for (int u = 0; u < VU; ++u)
#pragma unroll
      for (int x = 0; x < 2; ++x)
        dyn[(warp * BM + m) * (OS / 4) + ((8 * u + 2 * t + x) ^ (m & 7))] =
            make_float4(o[4 * u][2 * y + x], o[4 * u + 1][2 * y + x], o[4 * u + 2][2 * y + x], o[4 * u + 3][2 * y + x]);
  }
  __syncthreads();
  if (tid < BM) {
    float M = -INFINITY;
#pragma unroll
    for (int k = 0; k < NW; ++k) M = fmaxf(M, warp_ml[k][tid].x);
    const float at = M == -INFINITY ? 0.f : M;
    float L = 0.f;
#pragma unroll
    for (int k = 0; k < NW; ++k) {
      const float f = ex2(warp_ml[k][tid].x - at);
      factor[k][tid] = f;
      L = fmaf(warp_ml[k][tid].y, f, L);
    }
    joined[tid] = make_float2(M, L);
  }
  __syncthreads();
  const bool direct = !prefix && a.o_splits == 0;
  const int64_t all = (int64_t)a.rows * a.kv_heads * nG;
  for (int x = tid; x < BM * (D >> 2); x += NT) {
    const int mm = x / (D >> 2), c = x - mm * (D >> 2), m = m0 + mm;
    if (m >= rows_m) break;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < NW; ++k) {
      const float4 y = dyn[(k * BM + mm) * (OS / 4) + (c ^ (mm & 7))];
      const float f = factor[k][mm];
      v.x = fmaf(y.x, f, v.x);
      v.y = fmaf(y.y, f, v.y);
      v.z = fmaf(y.z, f, v.z);
      v.w = fmaf(y.w, f, v.w);
    }
    const float2 ml = joined[mm];
    const int r = prefix ? m / nG : r_own, mr = prefix ? m - r * nG : m;
    const int64_t idx = ((int64_t)r * a.kv_heads + h) * nG + mr;
    if (direct) {
      const float inv = ml.y == 0.f ? 0.f : 1.f / ml.y;
      const int i = mr / a.group;
      float* out = static_cast<float*>(a.out) + (((int64_t)r * a.n + i) * a.heads + h * a.group + mr - i * a.group) * D;
      reinterpret_cast<float4*>(out)[c] = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
      if (a.lse && c == 0) a.lse[idx] = ml.y == 0.f ? INFINITY : ml.x + log2f(ml.y);
    } else {
      const int64_t at = (int64_t)split * all + (prefix ? prefix_index(a, r, h, mr) : idx);
      reinterpret_cast<float4*>((prefix ? a.prefix_o : a.part_o) + at * D)[c] = v;
      if (c == 0) (prefix ? a.prefix_ml : a.part_ml)[at] = ml;
    }
  }
  if (a.status && !prefix && tid == 0 && blockIdx.x == 0 && h == 0) {
    const int e = a.lengths ? a.lengths[r_own] : a.capacity, s = a.starts ? a.starts[r_own] : 0;
    a.status[r_own] = (e < 0 || e > a.capacity || s < 0 || s > max(e, 0)) ? 8 : 0;
  }
}

template <int DC, bool FULL> cudaError_t launch(const AttnArgs& a, bool prefix, cudaStream_t stream) {
  const int64_t rows_m = (int64_t)(prefix ? a.rows : 1) * a.n * a.group;
  const int64_t S = prefix ? a.p_splits : (a.o_splits ? a.o_splits : 1);
  const dim3 grid((unsigned)((rows_m + BM - 1) / BM * S), (unsigned)(prefix ? a.kv_heads : a.rows * a.kv_heads));
  constexpr size_t smem = sizeof(float) * NW * BM * 64 * DC;
  const cudaError_t e = allow_smem<attn_f32_kernel<DC, FULL>>(smem);
  if (e != cudaSuccess) return e;
  attn_f32_kernel<DC, FULL><<<grid, NT, smem, stream>>>(a, prefix);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_attn_f32(const AttnArgs& a, bool prefix, cudaStream_t stream) {
  if (a.dim == 128) return launch<2, true>(a, prefix, stream);
  if (a.dim == 64) return launch<1, true>(a, prefix, stream);
  return a.dim < 64 ? launch<1, false>(a, prefix, stream) : launch<2, false>(a, prefix, stream);
}

}  // namespace sv
