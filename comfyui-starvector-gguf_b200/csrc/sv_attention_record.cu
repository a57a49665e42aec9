// sv_attention_record.cu -- attention of few query rows per key/value head over the
// cache held in 4 bits (sv_record.cuh): single tokens and drafts, float16 / bfloat16, one
// pass over the records at memory speed.
//
// Mathematics.  Row m of a unit (cache row r, key/value head h, eight to 32 of its query rows):
// with a key's groups k_d = mid_g + scale_g (c_d - 8),
//   q . k = sum_g scale_g (sum_{d in g} q_d c_d - 8 sum_{d in g} q_d) + sum_g mid_g sum_{d in g} q_d.
// The codes are whole numbers below 16, which float16 holds exactly: a nibble masked out
// of a word is, read as float16, its subnormal c 2^-24 (or, four bits further up, c 2^-20:
// those dimensions' queries are divided by 16), so a key needs no arithmetic before the
// tensor core takes it.  The queries are brought into float16's upper range by a power of two
// per row, which loses nothing of a bfloat16.  The scales multiply the groups' sums in f32; the rest,
// sum_g (mid_g - 8 scale_g) times the queries' group sums, is one product more, whose A operand is the
// record's pairs as they lie (the group sums in two halves).  So scores are as exact as those of f32 keys.
// Values are formed in float16, v = scale (c - 8) + mid rounded once, and the weights rounded to
// float16, for float16 outputs in two halves: one such rounding is about what the output's own adds (error of
// one token's output 0.0003 against 64 bits, 0.0002 that of the output's rounding alone; with both 0.00032).
// The softmax as in sv_attention_token.cu: the reference moves only when a score exceeds it by
// 2^8.
//
// Both products are turned round, S^T = K Q^T and O^T = V^T P^T (mma.m16n8k16): slots and
// dimensions fill the 16 rows, and the query rows take columns in eights, so that four heads of
// a group do not pay for sixteen; weights pass from the one to the other by a transposition
// (movmatrix).
//
// What bounds it: the records' bytes; next to that the instructions that turn codes into
// operands (about 270 per 16 slots and warp at eight rows; the memory's rate allows 450).  A warp
// takes tiles of 16 slots through a ring in shared memory of its own (cp.async, zeros for
// slots past the end): registers alone would keep too few bytes in flight, since 16 slots are
// only 2560.  Rows of a tile are taken in an order in which neither the keys' nor the
// values' reads meet in a bank (kSlot).
//
// Work split and joins as in sv_attention_token.cu: one list of chunks (a tile per warp) over all
// units, cut into equal parts, one per block; the last block to arrive joins a unit that
// several share, in block order.
#include <type_traits>

#include "sv_attention.h"
#include "sv_record.cuh"

namespace sv {
namespace {

constexpr int TK = 16;         // slots per tile
constexpr int kJoin = 16;      // parts per first-level group
constexpr int kMaxFlat = 32;   // parts joined in one level
constexpr float kSlack = 8.f;  // log2 by which a score may exceed its reference

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// d = a b + c; d = a b.
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1, const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  const float zero[4] = {0.f, 0.f, 0.f, 0.f};
  mma16(d, a0, a1, a2, a3, b0, b1, zero);
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t fma16(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t add16(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy16_or_zeros(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ unsigned arrive(unsigned* counter) {
  unsigned old;
  asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(old) : "l"(counter) : "memory");
  return old;
}

// The slot of a tile that row k of its products stands for: slots 4 (or 12) apart side by side, so
// that a quarter warp's 64-byte rows of 80-byte records fall into all banks once, and the
// values' rows 0, 2, 4, 6 into every second pair of them.
__device__ __forceinline__ int slot_at(int k) {
  constexpr uint64_t order = 0xBF9D7351AE8C6240ull;  // 0 4 2 6 12 8 14 10, then each + 1
  return (int)(order >> (4 * k)) & 15;
}

// Numbers of a record's layout for NI blocks of 32 dimensions.
template <int NI> struct Form {
  static constexpr int REC = 16 * NI + 16;                    // bytes
  static constexpr int NG = NI > 2 ? NI : 2 * NI;             // groups
  static constexpr int NB = NI > 2 ? 2 : 1;                   // words of a value that one thread turns into operands
  static constexpr int TILE = TK * REC;                       // bytes of a tile's keys (or values)
  static constexpr int COPIES = 2 * TILE / 512;               // 16-byte copies per thread and tile
};

// Like sv_attention_token.cu's: [a0, a1) the sinks before the window, [b0, b1) the rest.
struct RowTiles {
  int start, end, a0, a1, b0, b1, ta, tiles;
};

__device__ __noinline__ RowTiles row_tiles(const AttnArgs& a, int r) {
  RowTiles t;
  const RowSpan sp = row_span(a, r);
  t.start = sp.start;
  t.end = sp.end;
  t.b0 = window_low(a, sp.start, sp.end - a.n);
  t.b1 = max(sp.end, t.b0);
  t.a0 = sp.start;
  t.a1 = max(t.a0, min(sp.start + a.sinks, min(t.b0, t.b1)));
  t.ta = (t.a1 - t.a0 + TK - 1) / TK;
  t.tiles = max(1, t.ta + (t.b1 - t.b0 + TK - 1) / TK);
  return t;
}

// A place in the list of chunks: chunk k of unit (r, h), h counting the heads' groups of rows.
template <int NW> struct Place {
  int r, h, k, chunks;
  RowTiles rt;
  __device__ __forceinline__ void row(const AttnArgs& a, int r_) {
    r = r_;
    rt = row_tiles(a, r_);
    chunks = (rt.tiles + NW - 1) / NW;
  }
  // Whether the next place is another unit's.
  __device__ __forceinline__ bool next(const AttnArgs& a, int heads) {
    if (++k < chunks) return false;
    k = 0;
    if (++h == heads) {
      h = 0;
      if (r + 1 < a.rows) row(a, r + 1);  // (past the last chunk of all nothing is looked at)
    }
    return true;
  }
};

// NI blocks of 32 dimensions, NT column tiles of eight query rows, NW warps, a ring of RING tiles.
// MULTI: more than one query per row.
template <typename T, int NI, int NT, int NW, int RING, bool MULTI>
__global__ void __launch_bounds__(NW * 32, 1)
    attn_record_kernel(const __grid_constant__ AttnArgs a, const int blocks_max, const int row_groups) {
  using F = Form<NI>;
  constexpr int REC = F::REC, NG = F::NG, NB = F::NB, MT = 4 * NB, ROWS = 8 * NT, THREADS = NW * 32;
  constexpr int OS = 32 * NI;  // dimensions of the warps' outputs
  constexpr bool HALVES = std::is_same<T, __half>::value;
  constexpr uint32_t kOnes = 0x3c003c00u;
  extern __shared__ __align__(16) unsigned char ring_bytes[];  // [NW][RING][keys, values], then [NW][ROWS][OS] floats
  float* const outs = reinterpret_cast<float*>(ring_bytes + NW * RING * 2 * F::TILE);
  __shared__ float2 warp_ml[NW][ROWS];
  __shared__ float factor[kMaxFlat > NW ? kMaxFlat : NW][ROWS];
  __shared__ float2 part_ml[kMaxFlat][ROWS];
  __shared__ float2 joined[ROWS];
  __shared__ int scan[NW];
  __shared__ int sh_row, sh_before, sh_last[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int group = a.group, nG = MULTI ? a.n * group : group, K = a.kv_heads * row_groups, D = a.dim;

  // The warps' outputs: 4 dimensions c of row m, placed so that the fragments' writes do not meet in a bank.
  auto vec_at = [&](int w, int m, int c) {
    return reinterpret_cast<float4*>(outs) + (w * ROWS + m) * (OS / 4) + (c ^ (m >> 1 & 3) ^ (OS >= 128 ? c >> 2 & 4 : 0));
  };

  // Chunks of all rows, every head of a row having as many: see sv_attention_token.cu.
  const int per = (a.rows + THREADS - 1) / THREADS, row0 = tid * per;
  int mine = 0;
  for (int x = row0; x < min(row0 + per, a.rows); ++x) mine += (row_tiles(a, x).tiles + NW - 1) / NW;
  int upto = mine;
#pragma unroll
  for (int k = 1; k < 32; k <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, upto, k);
    if (lane >= k) upto += x;
  }
  if (lane == 31) scan[warp] = upto;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int k = 0; k < NW; ++k) {
    if (k == warp) upto += total;
    total += scan[k];
  }
  const int W = total * K;  // fits 31 bits (checked by the host)
  const int N = min(blocks_max, W), share = W / N, extra = W - share * N;
  const int c = blockIdx.x;
  if (c >= N) return;
  auto first_chunk = [&](int b) { return b * share + min(b, extra); };
  auto block_of = [&](int chunk) {
    const int b = chunk / (share + 1);
    return b < extra ? b : extra + (chunk - extra * (share + 1)) / share;
  };
  const int c0 = first_chunk(c), c1 = first_chunk(c + 1);
  if ((upto - mine) * K <= c0 && c0 < upto * K) {
    int x = row0, at = upto - mine;
    for (;; ++x) {
      const int chunks = (row_tiles(a, x).tiles + NW - 1) / NW;
      if (c0 < (at + chunks) * K) break;
      at += chunks;
    }
    sh_row = x;
    sh_before = at;
  }
  __syncthreads();
  Place<NW> p;
  p.row(a, sh_row);
  {
    const int off = c0 - sh_before * K;
    p.h = off / p.chunks;
    p.k = off - p.h * p.chunks;
  }
  int before = sh_before;  // chunks (of one head) before row p.r

  // ---- copies: this warp's tile of chunk f, the f-th place ahead
  Place<NW> f = p;
  int fetched = c0;
  const unsigned char *fk, *fv;  // its unit's records
  auto open = [&]() {
    const int64_t base = f.r * a.kv_row + (f.h / row_groups) * a.kv_head;
    fk = static_cast<const unsigned char*>(a.k) + base;
    fv = static_cast<const unsigned char*>(a.v) + base;
  };
  open();
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(ring_bytes) + warp * RING * 2 * F::TILE;
  uint32_t put = ring + lane * 16;
  const bool dense = a.kv_slot == REC;
  auto fetch = [&]() {
    if (fetched < c1) {
      const int tile = f.k * NW + warp;
      const bool in_a = tile < f.rt.ta;
      const int j0 = in_a ? f.rt.a0 + tile * TK : f.rt.b0 + (tile - f.rt.ta) * TK;
      const int count = tile < f.rt.tiles ? min(TK, (in_a ? f.rt.a1 : f.rt.b1) - j0) : 0;
      const int64_t off = j0 * a.kv_slot;
      if (dense && count == TK) {  // a run of bytes each
        const unsigned char *kb = fk + off + lane * 16, *vb = fv + off + lane * 16 - F::TILE;
#pragma unroll
        for (int x = 0; x < F::COPIES; ++x) {
          constexpr int K = F::TILE / 16;  // copies of keys
          const unsigned char* src = 32 * x + 32 <= K ? kb : 32 * x >= K ? vb : lane + 32 * x < K ? kb : vb;
          copy16(put + x * 512, src + x * 512);
        }
      } else if (count > 0) {
#pragma unroll 1
        for (int x = lane; x < 2 * F::TILE / 16; x += 32) {
          const int in = x >= F::TILE / 16 ? x - F::TILE / 16 : x, slot = in / (REC / 16);
          const int64_t at = off + slot * a.kv_slot + (in - slot * (REC / 16)) * 16;
          copy16_or_zeros(put + (x - lane) * 16, (x == in ? fk : fv) + (slot < count ? at : 0), slot < count);
        }
      }
      put = put + 2 * F::TILE == ring + lane * 16 + RING * 2 * F::TILE ? ring + lane * 16 : put + 2 * F::TILE;
      ++fetched;
      if (f.next(a, K)) open();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  // ---- queries: the B operand of each step over 16 dimensions, the groups' sums in halves, the rows' factors
  uint32_t qb[NT][NI][2][2], qm[NT][2];
  float fr[NT][2];
  auto load_q = [&](int r, int h) {
    const int head = h / row_groups, m0 = (h - head * row_groups) * ROWS;
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const int m = m0 + 8 * u + g, i = MULTI ? m / group : 0;
      const T* src = static_cast<const T*>(a.q) + r * a.q_row + i * a.q_tok + (int64_t)(head * group + m - i * group) * a.q_head;
      float x[NI][2][4], most = 0.f;
#pragma unroll
      for (int b = 0; b < NI; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int d = 32 * b + 16 * e + 4 * t;
          uint2 w = make_uint2(0u, 0u);
          if (m < nG && d < D) w = __ldg(reinterpret_cast<const uint2*>(src + d));
          const T* y = reinterpret_cast<const T*>(&w);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            x[b][e][k] = (float)y[k];
            if (fabsf(x[b][e][k]) < INFINITY) most = fmaxf(most, fabsf(x[b][e][k]));
          }
        }
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      // The row's largest value to [2^14, 2^15).
      const int ex = max(15, (int)(__float_as_uint(most) >> 23));
      const float up = copysignf(__uint_as_float((uint32_t)(268 - min(ex, 254)) << 23), a.scale);
      float sum[NG];
#pragma unroll
      for (int k = 0; k < NG; ++k) sum[k] = 0.f;
#pragma unroll
      for (int b = 0; b < NI; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            x[b][e][k] *= up;
            sum[NI > 2 ? b : 2 * b + e] += x[b][e][k];
          }
          qb[u][b][e][0] = pack16(x[b][e][0], x[b][e][1]);
          qb[u][b][e][1] = pack16(x[b][e][2] * 0.0625f, x[b][e][3] * 0.0625f);
        }
      // Group t's sum, in the keys' units; in halves, for scale (times -8) and mid.
      float own = 0.f;
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 1);
        sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 2);
        if (k == t) own = sum[k] * 0x1p-24f;
      }
      const float high = __half2float(__float2half_rn(own));
      qm[u][0] = pack16(-8.f * high, high);
      qm[u][1] = pack16(-8.f * (own - high), own - high);
      // (Scores past f32's range stay within it by a smaller factor: any of them is the whole softmax.  A
      // factor of zero would make NaN of hidden slots' -infinity.)
      const float mine = fmaxf(fabsf(a.scale) * __uint_as_float((uint32_t)(min(ex, 230) + 10) << 23), 0x1p-126f);  // 2^(ex - 141 + 24)
#pragma unroll
      for (int y = 0; y < 2; ++y) fr[u][y] = __shfl_sync(0xffffffffu, mine, 8 * t + 4 * y);
    }
  };

  auto write_out = [&](int r, int head, int m, int d, float4 x, float L) {  // m: row of the head's nG
    if (d >= D) return;
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const int i = MULTI ? m / group : 0;
    T* out = static_cast<T*>(a.out) + (((int64_t)r * a.n + i) * a.heads + head * group + m - i * group) * D + d;
    T y[4] = {from_float<T>(x.x * inv), from_float<T>(x.y * inv), from_float<T>(x.z * inv), from_float<T>(x.w * inv)};
    *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(y);
  };
  auto write_lse = [&](int r, int head, int m, float2 j) {
    if (a.lse) a.lse[(int64_t)(r * a.kv_heads + head) * nG + m] = j.y == 0.f ? INFINITY : j.x + log2f(j.y);
  };

  // The units this block shares with others: the one it starts in and the one it ends in at most.
  struct Shared { int r, h, first, end; };
  Shared shared_part[2];
  int shared_parts = 0;
  constexpr int VECS = ROWS * (OS / 4), ITEMS = (VECS + THREADS - 1) / THREADS;

#pragma unroll
  for (int k = 0; k < RING - 1; ++k) fetch();
  int at = c0;
  uint32_t get = ring;
  for (;;) {  // units
    load_q(p.r, p.h);
    const int head = p.h / row_groups, m0 = (p.h - head * row_groups) * ROWS, rows_here = min(ROWS, nG - m0);
    const int first = before * K + p.h * p.chunks, end = first + p.chunks, stop = min(end, c1);
    const RowTiles rt = p.rt;
    const int pos_first = rt.end - a.n, low_last = window_low(a, rt.start, rt.end - 1);
    // ref: a row's reference; edge: the raw score past which it moves.
    float o[NT][MT][4], ref[NT][2], edge[NT][2], l[NT][4];
#pragma unroll
    for (int u = 0; u < NT; ++u) {
#pragma unroll
      for (int y = 0; y < 2; ++y) ref[u][y] = edge[u][y] = -INFINITY;
#pragma unroll
      for (int k = 0; k < 4; ++k) l[u][k] = 0.f;
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[u][j][k] = 0.f;
    }
    for (; at < stop; ++at) {
      const int tile = (at - first) * NW + warp;
      const uint32_t kt = get, vt = kt + F::TILE;
      get = get + 2 * F::TILE == ring + RING * 2 * F::TILE ? ring : get + 2 * F::TILE;
      asm volatile("cp.async.wait_group %0;" ::"n"(RING - 2) : "memory");
      __syncwarp();
      fetch();  // into the place that the last round has left
      const bool in_a = tile < rt.ta;
      const int j0 = in_a ? rt.a0 + tile * TK : rt.b0 + (tile - rt.ta) * TK, jend = in_a ? rt.a1 : rt.b1;
      if (tile >= rt.tiles || j0 >= jend) continue;
      // ---- scores
      const int s0 = slot_at(g), s1 = slot_at(g + 8);
      float s[NT][4];  // slots s0 and s1 of rows 2 t and 2 t + 1, in units of 1 / fr
      {
        uint32_t kw[2][NI], pr[2][4], own[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t rec = kt + (x ? s1 : s0) * REC;
          if constexpr (NI == 4) {
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(kw[x][0]), "=r"(kw[x][1]), "=r"(kw[x][2]), "=r"(kw[x][3]) : "r"(rec + t * 16));
          } else if constexpr (NI == 2) {
            asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(kw[x][0]), "=r"(kw[x][1]) : "r"(rec + t * 8));
          } else {
#pragma unroll
            for (int b = 0; b < NI; ++b) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(kw[x][b]) : "r"(rec + (t * NI + b) * 4));
          }
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(pr[x][0]), "=r"(pr[x][1]), "=r"(pr[x][2]), "=r"(pr[x][3]) : "r"(rec + 16 * NI));
          asm volatile("ld.shared.u32 %0, [%1];" : "=r"(own[x]) : "r"(rec + 16 * NI + 4 * t));
        }
#pragma unroll
        for (int u = 0; u < NT; ++u) mma16(s[u], own[0], own[1], own[0], own[1], qm[u][0], qm[u][1]);
#pragma unroll
        for (int grp = 0; grp < NG; ++grp) {
          float acc[NT][4];
#pragma unroll
          for (int e = NI > 2 ? 0 : grp & 1; e < (NI > 2 ? 2 : (grp & 1) + 1); ++e) {
            const int b = NI > 2 ? grp : grp >> 1;
            const uint32_t w0 = e ? kw[0][b] >> 8 : kw[0][b], w1 = e ? kw[1][b] >> 8 : kw[1][b];
#pragma unroll
            for (int u = 0; u < NT; ++u) {
              if (NI > 2 && e)
                mma16(acc[u], w0 & 0x000f000fu, w1 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x00f000f0u, qb[u][b][e][0], qb[u][b][e][1], acc[u]);
              else
                mma16(acc[u], w0 & 0x000f000fu, w1 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x00f000f0u, qb[u][b][e][0], qb[u][b][e][1]);
            }
          }
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float sc = __low2float(*reinterpret_cast<const __half2*>(&pr[x][grp]));
#pragma unroll
            for (int u = 0; u < NT; ++u)
#pragma unroll
              for (int y = 0; y < 2; ++y) s[u][2 * x + y] = fmaf(sc, acc[u][2 * x + y], s[u][2 * x + y]);
          }
        }
      }
      const bool whole = j0 + TK <= jend && (in_a || !MULTI || (j0 >= low_last && j0 + TK - 1 <= pos_first));
      if (!whole) {
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int pos = MULTI ? pos_first + (m0 + 8 * u + 2 * t + y) / group : pos_first;
            const int low = window_low(a, rt.start, pos);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int j = j0 + (x ? s1 : s0);
              if (j >= jend || !slot_seen(a, rt.start, pos, low, j)) s[u][2 * x + y] = -INFINITY;
            }
          }
      }
      if (a.scores) {
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const int j = j0 + (x ? s1 : s0), m = 8 * u + 2 * t + y;
              if (j < jend && m < rows_here)
                a.scores[((int64_t)(p.r * a.kv_heads + head) * nG + m0 + m) * a.capacity + j] = s[u][2 * x + y] * fr[u][y];
            }
      }
      // ---- weights
      bool over = false;
#pragma unroll
      for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int y = 0; y < 2; ++y) over |= fmaxf(s[u][y], s[u][2 + y]) > edge[u][y];
      if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            float mx = fmaxf(s[u][y], s[u][2 + y]);
#pragma unroll
            for (int k = 4; k < 32; k <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
            const float now = fmaxf(mx * fr[u][y], ref[u][y]);
            const float by = now == ref[u][y] ? 1.f : ex2(ref[u][y] - now);
            ref[u][y] = now;
            edge[u][y] = now == -INFINITY ? -INFINITY : (now + kSlack) / fr[u][y];
            l[u][y] *= by;
            l[u][2 + y] *= by;
#pragma unroll
            for (int j = 0; j < MT; ++j) {
              o[u][j][y] *= by;
              o[u][j][2 + y] *= by;
            }
          }
      }
      // Weights as B operand: slots of rows 0..7 and 8..15 of the tile's order; their sums are a product with ones.
      uint32_t pb[NT][2];
      [[maybe_unused]] uint32_t pl[NT][2];  // float16 outputs: what the rounding left
#pragma unroll
      for (int u = 0; u < NT; ++u) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float w[2];
#pragma unroll
          for (int y = 0; y < 2; ++y) w[y] = ex2(fmaf(s[u][2 * x + y], fr[u][y], -(ref[u][y] == -INFINITY ? 0.f : ref[u][y])));
          const uint32_t both = pack16(w[0], w[1]);
          pb[u][x] = transposed(both);
          if constexpr (HALVES) {
            const float2 high = __half22float2(*reinterpret_cast<const __half2*>(&both));
            pl[u][x] = transposed(pack16(w[0] - high.x, w[1] - high.y));
          }
        }
        mma16(l[u], kOnes, kOnes, kOnes, kOnes, pb[u][0], pb[u][1], l[u]);
        if constexpr (HALVES) mma16(l[u], kOnes, kOnes, kOnes, kOnes, pl[u][0], pl[u][1], l[u]);
      }
      // ---- values
      {
        const int va = slot_at(2 * t), vb = slot_at(2 * t + 1);  // and each + 1 in rows 8..15
        const uint32_t ra[4] = {vt + va * REC, vt + vb * REC, vt + (va + 1) * REC, vt + (vb + 1) * REC};
        uint32_t vw[4][NB], pr[4][2];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if constexpr (NI == 4) {
            asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(vw[x][0]), "=r"(vw[x][1]) : "r"(ra[x] + g * 8));
            asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(pr[x][0]), "=r"(pr[x][1]) : "r"(ra[x] + 16 * NI + (g & 1) * 8));
          } else if constexpr (NI == 3) {  // words 2 g, 2 g + 1 of twelve
            const int w = min(2 * g, 10);
            asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(vw[x][0]), "=r"(vw[x][1]) : "r"(ra[x] + w * 4));
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(pr[x][0]) : "r"(ra[x] + 16 * NI + w % 3 * 4));
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(pr[x][1]) : "r"(ra[x] + 16 * NI + (w + 1) % 3 * 4));
          } else {
            const int w = NI == 2 ? g : g & 3;
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(vw[x][0]) : "r"(ra[x] + w * 4));
            asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(pr[x][0]), "=r"(pr[x][1]) : "r"(ra[x] + 16 * NI + w % NI * 8));
          }
        }
        uint32_t sc[2][2], mi[2][2];  // [rows 0..7, 8..15][group]
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            sc[x][k] = __byte_perm(pr[2 * x][k], pr[2 * x + 1][k], 0x5410);
            mi[x][k] = __byte_perm(pr[2 * x][k], pr[2 * x + 1][k], 0x7632);
          }
        // A group that stands for NaN must not reach the rows that do not see its slot (0 * NaN): the
        // product takes zeros in its place, and the rows that see it become NaN below.
        bool hide = false;
        uint32_t bad[2][2] = {{0u, 0u}, {0u, 0u}};
        if (MULTI && !whole) {
          uint32_t any = 0u;
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const uint32_t lo = (sc[x][k] & 0x7c00u) == 0x7c00u || (mi[x][k] & 0x7c00u) == 0x7c00u ? 0xffffu : 0u;
              const uint32_t hi = (sc[x][k] & 0x7c000000u) == 0x7c000000u || (mi[x][k] & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u;
              bad[x][k] = lo | hi;
              any |= bad[x][k];
            }
          hide = __any_sync(0xffffffffu, any != 0u);
          if (hide) {
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
              for (int k = 0; k < 2; ++k) sc[x][k] &= ~bad[x][k], mi[x][k] &= ~bad[x][k];
          }
        }
        // The value of nibble j (0..3) of a 16-bit half, of two slots side by side.
        auto value = [&](uint32_t w, int j, uint32_t scale, uint32_t mid) {
          const uint32_t x = j & 2 ? w >> 8 : w;
          const uint32_t c8 = j & 1 ? fma16((x & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, 0xd480d480u)   // (1024 + 16 c) / 16 - 72
                                    : add16((x & 0x000f000fu) | 0x64006400u, 0xe408e408u);              // 1024 + c - 1032
          return fma16(c8, scale, mid);
        };
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const uint32_t l0 = __byte_perm(vw[0][b], vw[1][b], 0x5410), h0 = __byte_perm(vw[0][b], vw[1][b], 0x7632);
          const uint32_t l1 = __byte_perm(vw[2][b], vw[3][b], 0x5410), h1 = __byte_perm(vw[2][b], vw[3][b], 0x7632);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int k = NI > 2 ? b : j >> 1;
            const uint32_t a0 = value(l0, j, sc[0][k], mi[0][k]), a1 = value(h0, j, sc[0][k], mi[0][k]);
            const uint32_t a2 = value(l1, j, sc[1][k], mi[1][k]), a3 = value(h1, j, sc[1][k], mi[1][k]);
#pragma unroll
            for (int u = 0; u < NT; ++u) {
              mma16(o[u][4 * b + j], a0, a1, a2, a3, pb[u][0], pb[u][1], o[u][4 * b + j]);
              if constexpr (HALVES) mma16(o[u][4 * b + j], a0, a1, a2, a3, pl[u][0], pl[u][1], o[u][4 * b + j]);
            }
          }
        }
        if (MULTI && hide) {
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int k = NI > 2 ? b : j >> 1;
              const uint32_t x = bad[0][k] & 0x3c003c00u, z = bad[1][k] & 0x3c003c00u;
#pragma unroll
              for (int u = 0; u < NT; ++u) {
                float seen[4];
                mma16(seen, x, x, z, z, pb[u][0], pb[u][1]);
#pragma unroll
                for (int q = 0; q < 4; ++q)
                  if (seen[q] != 0.f) o[u][4 * b + j][q] = __int_as_float(0x7fc00000);
              }
            }
        }
      }
    }

    // ---- the warps' results into shared memory
#pragma unroll
    for (int u = 0; u < NT; ++u) {
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int m = 8 * u + 2 * t + y;
        if (g == 0) warp_ml[warp][m] = make_float2(ref[u][y], l[u][y]);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const int w = NI > 2 ? 2 * g + b : g, tw = w / NI, blk = w - tw * NI;
          if (tw < 4) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int j = 4 * b + 2 * e;
              *vec_at(warp, m, 8 * blk + 4 * e + tw) = make_float4(o[u][j][y], o[u][j][2 + y], o[u][j + 1][y], o[u][j + 1][2 + y]);
            }
          }
        }
      }
    }
    __syncthreads();
    const bool alone = first >= c0 && end <= c1;
    const int slot = 2 * c + (first >= c0);
    if (tid < ROWS) {
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int k = 0; k < NW; ++k) M = fmaxf(M, warp_ml[k][tid].x);
      const float z = M == -INFINITY ? 0.f : M;
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        const float by = ex2(warp_ml[k][tid].x - z);
        factor[k][tid] = by;
        L = fmaf(warp_ml[k][tid].y, by, L);
      }
      joined[tid] = make_float2(M, L);
      if (tid < rows_here) {
        if (alone)
          write_lse(p.r, head, m0 + tid, joined[tid]);
        else
          a.part_ml[(int64_t)slot * ROWS + tid] = joined[tid];
      }
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < ITEMS; ++x) {
      const int v = tid + x * THREADS, m = v / (OS / 4), d = (v - m * (OS / 4)) * 4;
      if (m >= rows_here) continue;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        const float4 y = *vec_at(k, m, d >> 2);
        const float by = factor[k][m];
        sum.x = fmaf(y.x, by, sum.x);
        sum.y = fmaf(y.y, by, sum.y);
        sum.z = fmaf(y.z, by, sum.z);
        sum.w = fmaf(y.w, by, sum.w);
      }
      if (alone)
        write_out(p.r, head, m0 + m, d, sum, joined[m].y);
      else
        *reinterpret_cast<float4*>(a.part_o + ((int64_t)slot * ROWS + m) * OS + d) = sum;
    }
    if (!alone) shared_part[shared_parts++] = {p.r, p.h, first, end};
    if (a.status && tid == 0 && p.h == K - 1 && end <= c1) {
      const int e = a.lengths ? a.lengths[p.r] : a.capacity, s = a.starts ? a.starts[p.r] : 0;
      a.status[p.r] = (e < 0 || e > a.capacity || s < 0 || s > max(e, 0)) ? 8 : 0;
    }
    __syncthreads();
    if (end >= c1) break;
    p.k = 0;
    if (++p.h == K) {
      p.h = 0;
      before += p.chunks;
      p.row(a, p.r + 1);
    }
  }

  // ---- units shared with other blocks: who arrives last joins
  auto join = [&](const Shared& q, int c_first, int b0, int step, int count, bool last) {
    const int head = q.h / row_groups, m0 = (q.h - head * row_groups) * ROWS, rows_here = min(ROWS, nG - m0);
    auto slot_of = [&](int k) { return (int64_t)2 * (b0 + k * step) + (b0 + k * step == c_first); };
    __syncthreads();
    for (int x = tid; x < count * ROWS; x += THREADS) {
      const int k = x / ROWS, m = x - k * ROWS;
      if (m < rows_here) part_ml[k][m] = __ldcg(a.part_ml + slot_of(k) * ROWS + m);
    }
    __syncthreads();
    if (tid < rows_here) {
      float M = -INFINITY, L = 0.f;
      for (int k = 0; k < count; ++k) M = fmaxf(M, part_ml[k][tid].x);
      const float z = M == -INFINITY ? 0.f : M;
      for (int k = 0; k < count; ++k) {
        const float2 ml = part_ml[k][tid];
        const float by = ml.y == 0.f ? 0.f : ex2(ml.x - z);
        factor[k][tid] = by;
        L = fmaf(ml.y, by, L);
      }
      joined[tid] = make_float2(M, L);
      if (last)
        write_lse(q.r, head, m0 + tid, joined[tid]);
      else
        a.part_ml[slot_of(0) * ROWS + tid] = joined[tid];
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < ITEMS; ++x) {
      const int v = tid + x * THREADS, m = v / (OS / 4), d = (v - m * (OS / 4)) * 4;
      if (m >= rows_here) continue;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
      for (int k = 0; k < count; ++k) {
        const float4 y = __ldcg(reinterpret_cast<const float4*>(a.part_o + (slot_of(k) * ROWS + m) * OS + d));
        const float by = factor[k][m];
        sum.x = fmaf(y.x, by, sum.x);
        sum.y = fmaf(y.y, by, sum.y);
        sum.z = fmaf(y.z, by, sum.z);
        sum.w = fmaf(y.w, by, sum.w);
      }
      if (last)
        write_out(q.r, head, m0 + m, d, sum, joined[m].y);
      else
        *reinterpret_cast<float4*>(a.part_o + (slot_of(0) * ROWS + m) * OS + d) = sum;
    }
  };
  auto arrives_last = [&](unsigned* counter, int count) {
    const bool is_last = arrive(counter) == (unsigned)count - 1u;
    if (is_last) *counter = 0u;
    return is_last;
  };
  if (tid < shared_parts) {
    const Shared& q = shared_part[tid];
    const int c_first = block_of(q.first), parts = block_of(q.end - 1) - c_first + 1;
    const int b0 = c_first + (c - c_first) / kJoin * kJoin;
    sh_last[tid] = parts > kMaxFlat ? arrives_last(a.counters + (int64_t)a.rows * K + 2 * b0 + (b0 == c_first),
                                                   min(kJoin, c_first + parts - b0))
                                    : arrives_last(a.counters + q.r * K + q.h, parts);
  }
  __syncthreads();
  for (int x = 0; x < shared_parts; ++x) {
    if (!sh_last[x]) continue;
    const Shared q = shared_part[x];
    const int c_first = block_of(q.first), parts = block_of(q.end - 1) - c_first + 1;
    int step = 1, count = parts;
    if (parts > kMaxFlat) {
      const int b0 = c_first + (c - c_first) / kJoin * kJoin;
      join(q, c_first, b0, 1, min(kJoin, c_first + parts - b0), false);
      step = kJoin;
      count = (parts + kJoin - 1) / kJoin;
      __syncthreads();
      if (tid == 0) sh_last[x] = arrives_last(a.counters + q.r * K + q.h, count);
      __syncthreads();
      if (!sh_last[x]) continue;
    }
    join(q, c_first, c_first, step, count, true);
  }
}

template <typename T, int NI, int NT, int NW, int RING, bool MULTI>
cudaError_t record(const AttnArgs& a, int row_groups, cudaStream_t stream) {
  constexpr size_t smem = (size_t)NW * RING * 2 * Form<NI>::TILE + sizeof(float) * NW * 8 * NT * 32 * NI;
  const cudaError_t e = allow_smem<attn_record_kernel<T, NI, NT, NW, RING, MULTI>>(smem);
  if (e != cudaSuccess) return e;
  attn_record_kernel<T, NI, NT, NW, RING, MULTI><<<kTokenBlocks, NW * 32, smem, stream>>>(a, kTokenBlocks, row_groups);
  return cudaGetLastError();
}

template <typename T, int NI, bool MULTI> cudaError_t record_rows(const AttnArgs& a, const RecordRows& x, cudaStream_t stream) {
  if (x.tiles == 1) return record<T, NI, 1, 16, 3, MULTI>(a, x.groups, stream);
  return record<T, NI, 2, 8, 4, MULTI>(a, x.groups, stream);
}

template <typename T> cudaError_t record_any(const AttnArgs& a, const RecordRows& x, cudaStream_t stream) {
  auto dims = [&](auto multi) {
    constexpr bool M = decltype(multi)::value;
    if (a.dim > 96) return record_rows<T, 4, M>(a, x, stream);
    if (a.dim > 64) return record_rows<T, 3, M>(a, x, stream);
    return a.dim > 32 ? record_rows<T, 2, M>(a, x, stream) : record_rows<T, 1, M>(a, x, stream);
  };
  return a.n > 1 ? dims(std::true_type()) : dims(std::false_type());
}

}  // namespace

cudaError_t launch_attn_record(const AttnArgs& a, const RecordRows& x, cudaStream_t stream) {
  return a.dtype == 1 ? record_any<__half>(a, x, stream) : record_any<__nv_bfloat16>(a, x, stream);
}

}  // namespace sv
