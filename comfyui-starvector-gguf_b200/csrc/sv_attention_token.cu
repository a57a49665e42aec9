// sv_attention_token.cu -- attention of few query rows per key/value head over the
// cache: at most 16 rows (query, head of the group), so single tokens, and drafts of a few
// where the groups are small; float16 / bfloat16, one pass over the slots at memory speed.
//
// Mathematics.  Row m of a unit (cache row r, key/value head h): s_j = (q_m . k_j) *
// scale * log2 e, o = sum_j 2^(s_j - ref) v_j, l = sum_j 2^(s_j - ref), joined over
// slices of the slots by their references.  ref follows the running maximum only when
// a score exceeds it by more than 2^8: the weights stay below 2^8 (exact in f32, in
// range of float16), and most tiles need no maximum exchange and no rescaling.
//
// What bounds it: the bytes of the keys and values.  A warp takes 16 slots at a time
// straight from global memory into the fragments of mma.m16n8k16, without shared
// memory:
//   * scores = Q K^T: the sum over dimensions may run in any order, so a thread's
//     16-byte vector of a key (8 consecutive dimensions) serves as the B operand of
//     two products whose A operand takes the queries' vectors in the same order;
//   * output = P V: the thread that holds slots 2t, 2t+1, 2t+8, 2t+9 of the score
//     fragment loads those four slots' vectors of 8 dimensions and interleaves them in
//     pairs (byte permutes); which output column a dimension takes is free, so a
//     thread ends with 16 consecutive dimensions of its two rows.
// The next tile's keys are fetched as soon as the scores are formed, the next values
// after the product, so a warp keeps 4 to 8 KB in flight.
//
// Work split: the chunks (eight tiles, one per warp) of all units form one list, in unit
// order, cut into equal parts, one per block; ragged lengths balance by themselves.  A unit that spans
// several blocks leaves partial results, which the last block to arrive joins, in
// block order (so results repeat bit for bit); past 32 parts in two levels, so that no
// block joins more than a few dozen.  The sums' counters return to zero.
#include <type_traits>

#include "sv_attention.h"

namespace sv {
namespace {

constexpr int NW = kTokenWarps, NT = NW * 32;
constexpr int TK = 16;         // slots per tile
constexpr int kJoin = 16;      // parts per first-level group
constexpr int kMaxFlat = 32;   // parts joined in one level
constexpr float kSlack = 8.f;  // log2 by which a score may exceed its reference

template <typename T> struct Mma;
template <> struct Mma<__half> {
  __device__ static void run(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                             uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  __device__ static uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ static uint32_t not_finite(uint32_t w) {
    return (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u;
  }
  // The two values of a word, zeros for those that are not finite.
  __device__ static uint32_t finite(uint32_t w) {
    return ((w & 0x7c00u) == 0x7c00u ? 0u : w & 0xffffu) | ((w & 0x7c000000u) == 0x7c000000u ? 0u : w & 0xffff0000u);
  }
};
template <> struct Mma<__nv_bfloat16> {
  __device__ static void run(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                             uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  __device__ static uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ static uint32_t not_finite(uint32_t w) {
    return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
  }
  // The two values of a word, zeros for those that are not finite.
  __device__ static uint32_t finite(uint32_t w) {
    return ((w & 0x7f80u) == 0x7f80u ? 0u : w & 0xffffu) | ((w & 0x7f800000u) == 0x7f800000u ? 0u : w & 0xffff0000u);
  }
};

__device__ __forceinline__ uint4 load_stream(const void* p, bool ok) {
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (ok)
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
  return v;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Counts an arrival: what the block wrote before (ordered by a barrier) is visible to
// who arrives later, and this thread sees what earlier ones wrote.
__device__ __forceinline__ unsigned arrive(unsigned* counter) {
  unsigned old;
  asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(old) : "l"(counter) : "memory");
  return old;
}

// What one row's tiles are: [a0, a1) the sinks before the window, [b0, b1) the rest.
struct RowTiles {
  int start, end, a0, a1, b0, b1, ta, tiles;
  __device__ int chunks() const { return (tiles + NW - 1) / NW; }
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
  t.tiles = max(1, t.ta + (t.b1 - t.b0 + TK - 1) / TK);  // an empty row is a tile of nothing
  return t;
}

// One block's part of a unit (row r, head h): tiles [t0, t1) of the row.
struct Part {
  int r, h, before, first, end, t0, t1;  // before, first, end: chunks before the row (one head), of the unit
  RowTiles rt;
  __device__ __forceinline__ void open(int K, int c0, int c1) {
    first = before * K + h * rt.chunks();
    end = first + rt.chunks();
    t0 = (max(c0, first) - first) * NW;
    t1 = min(rt.tiles, (c1 - first) * NW);
  }
};

// MULTI: more than one query per row (then a tile may be visible to some of them only).
extern __shared__ float dyn[];  // [NW][16][64 DC]
template <typename T, int DC, bool FULL, bool MULTI>
__global__ void __launch_bounds__(NT, kTokenPerSM) attn_token_kernel(const __grid_constant__ AttnArgs a, const int blocks_max) {
  // The warps' outputs in shared memory: 16-byte vector c of row m, placed so that neither
  // the fragments' writes nor the rows' reads meet in a bank.
  constexpr int OS = DC * 64;
  auto vec_at = [](int w, int m, int c) {
    return reinterpret_cast<float4*>(dyn) + (w * 16 + m) * (OS / 4) + (c ^ (m & 1) ^ ((c >> 2) & 2));
  };
  __shared__ float2 warp_ml[NW][16];
  __shared__ float factor[kMaxFlat * 2][16];
  __shared__ float2 part_ml[kMaxFlat * 2][16];
  __shared__ float2 joined[16];
  __shared__ int scan[NW];
  __shared__ int sh_row, sh_before, sh_last[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int group = a.group, nG = MULTI ? a.n * group : group, K = a.kv_heads, D = FULL ? 64 * DC : a.dim;
  const int vecs = D >> 3;

  // Chunks (a tile per warp) of all rows, every head of a row having as many: thread x counts rows
  // [x per, (x + 1) per), a scan gives the total and what lies before each thread.
  const int per = (a.rows + NT - 1) / NT, row0 = tid * per;
  int mine = 0;
  for (int x = row0; x < min(row0 + per, a.rows); ++x) mine += row_tiles(a, x).chunks();
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
  // Blocks in use (a short call takes one per chunk); the first `extra` take one chunk more.
  const int N = min(blocks_max, W), share = W / N, extra = W - share * N;
  const int c = blockIdx.x;
  launch_dependents();
  if (c >= N) {
    wait_before();
    return;
  }
  auto first_chunk = [&](int b) { return b * share + min(b, extra); };
  auto block_of = [&](int chunk) {
    const int b = chunk / (share + 1);
    return b < extra ? b : extra + (chunk - extra * (share + 1)) / share;
  };
  const int c0 = first_chunk(c), c1 = first_chunk(c + 1);
  // The row that holds chunk c0, and the chunks (of one head) before it.
  if ((upto - mine) * K <= c0 && c0 < upto * K) {
    int x = row0, at = upto - mine;
    for (;; ++x) {
      const int chunks = row_tiles(a, x).chunks();
      if (c0 < (at + chunks) * K) break;
      at += chunks;
    }
    sh_row = x;
    sh_before = at;
  }
  __syncthreads();
  Part p;
  p.r = sh_row;
  p.before = sh_before;
  p.rt = row_tiles(a, p.r);
  p.h = (c0 - p.before * K) / p.rt.chunks();
  p.open(K, c0, c1);
  const int64_t all_rows = (int64_t)a.rows * K * nG;
  const int row_vecs = D >> 2;

  // Queries of rows g and g + 8, vectors t, t + 4, ...
  uint4 qf[2][2 * DC], kf[2][2 * DC], vf[4][DC];
  auto load_q = [&](const Part& p) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int m = g + 8 * x, i = MULTI ? m / group : 0, hd = p.h * group + m - i * group;
      const T* src = static_cast<const T*>(a.q) + p.r * a.q_row + i * a.q_tok + hd * a.q_head;
#pragma unroll
      for (int u = 0; u < 2 * DC; ++u) {
        const int vec = 4 * u + t;
        qf[x][u] = m < nG && (FULL || vec < vecs) ? __ldg(reinterpret_cast<const uint4*>(src) + vec)
                                                  : make_uint4(0u, 0u, 0u, 0u);
      }
    }
  };
  // The next tile to fetch: its slots [fetch_j0, fetch_end) and its unit's offset.
  int fetch_j0, fetch_end;
  int64_t fetch_base;
  auto tile_at = [&](const RowTiles& rt, int tile, int& j0, int& jend) {
    const bool in_a = tile < rt.ta;
    j0 = in_a ? rt.a0 + tile * TK : rt.b0 + (tile - rt.ta) * TK;
    jend = in_a ? rt.a1 : rt.b1;
  };
  auto fetch_at = [&](const Part& p, int tile) {
    tile_at(p.rt, tile, fetch_j0, fetch_end);
    if (tile >= p.t1) fetch_end = 0;
    fetch_base = p.r * a.kv_row + p.h * a.kv_head;
  };
  auto load_k = [&]() {
    const T* base = static_cast<const T*>(a.k) + fetch_base + t * 8;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int j = fetch_j0 + 8 * x + g;
      const T* src = base + j * a.kv_slot;
#pragma unroll
      for (int u = 0; u < 2 * DC; ++u)
        kf[x][u] = load_stream(src + 32 * u, j < fetch_end && (FULL || 4 * u + t < vecs));
    }
  };
  auto load_v = [&]() {
    const T* base = static_cast<const T*>(a.v) + fetch_base + g * 8;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int j = fetch_j0 + 2 * t + (x & 1) + (x >> 1) * 8;
      const T* src = base + j * a.kv_slot;
#pragma unroll
      for (int u = 0; u < DC; ++u)
        vf[x][u] = load_stream(src + 64 * u, j < fetch_end && (FULL || 8 * u + g < vecs));
    }
  };
  auto write_out = [&](const Part& p, int m, int d, float4 x, float L) {
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const int i = MULTI ? m / group : 0;
    T* out = static_cast<T*>(a.out) + (((int64_t)p.r * a.n + i) * a.heads + p.h * group + m - i * group) * D + d;
    *reinterpret_cast<uint2*>(out) =
        make_uint2(Mma<T>::pack(x.x * inv, x.y * inv), Mma<T>::pack(x.z * inv, x.w * inv));
  };
  auto write_lse = [&](const Part& p, int m) {
    if (a.lse)
      a.lse[(int64_t)(p.r * K + p.h) * nG + m] =
          joined[m].y == 0.f ? INFINITY : joined[m].x + log2f(joined[m].y);
  };
  // Joins `count` parts of a unit (and, `last`, the prefix's), the k-th that of block
  // b0 + k * step; c_first is the unit's first block.  ahead: the first parts' values are
  // fetched while the factors are made (where registers are free).
  auto join = [&](const Part& p, int c_first, int b0, int step, int count, bool last, auto ahead) {
    constexpr int ITEMS = (16 * DC * 16 + NT - 1) / NT, AHEAD = decltype(ahead)::value ? 6 : 0;
    const int more = last ? a.p_splits : 0, all_parts = count + more;
    if (more) wait_before();  // the prefix's kernel may have run beside this one
    const int64_t row0 = prefix_index(a, p.r, p.h, 0);
    auto slot_of = [&](int k) { return 2 * (b0 + k * step) + (b0 + k * step == c_first); };
    // Row m (of nG) and first dimension of this thread's x-th vector of four.
    int m[ITEMS], d[ITEMS];
#pragma unroll
    for (int x = 0; x < ITEMS; ++x) {
      m[x] = (tid + x * NT) / row_vecs;
      d[x] = (tid + x * NT - m[x] * row_vecs) * 4;
    }
    auto part_at = [&](int k, int x) {
      return __ldcg(reinterpret_cast<const float4*>(
          k < count ? a.part_o + ((int64_t)slot_of(k) * 16 + m[x]) * D + d[x]
                    : a.prefix_o + ((int64_t)(k - count) * all_rows + row0 + m[x]) * D + d[x]));
    };
    __syncthreads();
    float4 early[AHEAD ? AHEAD : 1][ITEMS];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
#pragma unroll
      for (int x = 0; x < ITEMS; ++x)
        if (k < all_parts && m[x] < nG) early[k][x] = part_at(k, x);
    for (int x = tid; x < all_parts * 16; x += NT) {
      const int k = x >> 4, mm = x & 15;
      if (mm < nG)
        part_ml[k][mm] = __ldcg(k < count ? a.part_ml + slot_of(k) * 16 + mm
                                          : a.prefix_ml + (int64_t)(k - count) * all_rows + row0 + mm);
    }
    __syncthreads();
    if (tid < nG) {
      float M = -INFINITY;
      for (int k = 0; k < all_parts; ++k) M = fmaxf(M, part_ml[k][tid].x);
      const float at = M == -INFINITY ? 0.f : M;
      float L = 0.f;
#pragma unroll 4
      for (int k = 0; k < all_parts; ++k) {
        const float2 ml = part_ml[k][tid];
        const float f = ml.y == 0.f ? 0.f : ex2(ml.x - at);
        factor[k][tid] = f;
        L = fmaf(ml.y, f, L);
      }
      joined[tid] = make_float2(M, L);
    }
    __syncthreads();
    float4 v[ITEMS];
#pragma unroll
    for (int x = 0; x < ITEMS; ++x) v[x] = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](int x, float4 y, float f) {
      v[x].x = fmaf(y.x, f, v[x].x);
      v[x].y = fmaf(y.y, f, v[x].y);
      v[x].z = fmaf(y.z, f, v[x].z);
      v[x].w = fmaf(y.w, f, v[x].w);
    };
#pragma unroll
    for (int x = 0; x < ITEMS; ++x) {
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
        if (k < all_parts && m[x] < nG) add(x, early[k][x], factor[k][m[x]]);
    }
#pragma unroll 4
    for (int k = AHEAD; k < all_parts; ++k)
#pragma unroll
      for (int x = 0; x < ITEMS; ++x)
        if (m[x] < nG) add(x, part_at(k, x), factor[k][m[x]]);
#pragma unroll
    for (int x = 0; x < ITEMS; ++x) {
      if (m[x] >= nG) continue;
      if (last)
        write_out(p, m[x], d[x], v[x], joined[m[x]].y);
      else
        *reinterpret_cast<float4*>(a.part_o + ((int64_t)slot_of(0) * 16 + m[x]) * D + d[x]) = v[x];
    }
    if (tid < nG) {
      if (last)
        write_lse(p, tid);
      else
        a.part_ml[slot_of(0) * 16 + tid] = joined[tid];
    }
  };

  // The units this block shares with others: the one it starts in and the one it ends
  // in at most.  They are joined at the end, when nothing is left to fetch.
  Part shared_part[2];
  int shared_parts = 0;
  load_q(p);
  fetch_at(p, p.t0 + warp);
  load_k();
  load_v();
  for (;;) {
    Part next = p;
    const bool more_units = p.end < c1;
    if (more_units) {
      if (++next.h == K) {
        next.h = 0;
        next.before += next.rt.chunks();
        next.rt = row_tiles(a, ++next.r);
      }
      next.open(K, c0, c1);
    }
    const int unit = p.r * K + p.h;
    int pos[2], low[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      pos[x] = MULTI ? p.rt.end - a.n + (g + 8 * x) / group : p.rt.end - 1;
      low[x] = window_low(a, p.rt.start, pos[x]);
    }
    const int pos_first = p.rt.end - a.n, low_last = window_low(a, p.rt.start, p.rt.end - 1);
    const T* vb = static_cast<const T*>(a.v) + p.r * a.kv_row + p.h * a.kv_head;
    float o[8 * DC][4];
#pragma unroll
    for (int j = 0; j < 8 * DC; ++j)
#pragma unroll
      for (int x = 0; x < 4; ++x) o[j][x] = 0.f;
    float ref[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    // A warp's last round fetches its first tile of the next unit.
    for (int tile = p.t0 + warp;; tile += NW) {
      const bool work = tile < p.t1, again = tile + NW < p.t1;
      if (again) {
        fetch_at(p, tile + NW);
      } else {
        fetch_at(next, next.t0 + warp);
        if (!more_units) fetch_end = 0;
      }
      int j0, jend;
      tile_at(p.rt, tile, j0, jend);
      float s[2][4];
      if (work) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int k = 0; k < 4; ++k) s[x][k] = 0.f;
#pragma unroll
        for (int u = 0; u < 2 * DC; ++u) {
          Mma<T>::run(s[x], qf[0][u].x, qf[1][u].x, qf[0][u].y, qf[1][u].y, kf[x][u].x, kf[x][u].y);
          Mma<T>::run(s[x], qf[0][u].z, qf[1][u].z, qf[0][u].w, qf[1][u].w, kf[x][u].z, kf[x][u].w);
        }
      }
      }
      load_k();
      if (work) {
      const bool whole = j0 + TK <= jend &&
                         (tile < p.rt.ta || !MULTI || (j0 >= low_last && j0 + TK - 1 <= pos_first));
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int k = 0; k < 4; ++k) s[x][k] *= a.scale;
      if (!whole) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int j = j0 + 8 * x + 2 * t + (k & 1), y = k >> 1;
            if (j >= jend || !slot_seen(a, p.rt.start, pos[y], low[y], j)) s[x][k] = -INFINITY;
          }
      }
      if (a.scores) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int j = j0 + 8 * x + 2 * t + (k & 1), m = g + 8 * (k >> 1);
            if (j < jend && m < nG) a.scores[((int64_t)unit * nG + m) * a.capacity + j] = s[x][k];
          }
      }
      float mx[2];
#pragma unroll
      for (int y = 0; y < 2; ++y)
        mx[y] = fmaxf(fmaxf(s[0][2 * y], s[0][2 * y + 1]), fmaxf(s[1][2 * y], s[1][2 * y + 1]));
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
          for (int j = 0; j < 8 * DC; ++j) {
            o[j][2 * y] *= f;
            o[j][2 * y + 1] *= f;
          }
        }
      }
      uint32_t w16[4];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const float at = ref[y] == -INFINITY ? 0.f : ref[y];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float p0 = ex2(s[x][2 * y] - at), p1 = ex2(s[x][2 * y + 1] - at);
          l[y] += p0 + p1;
          w16[2 * x + y] = Mma<T>::pack(p0, p1);
          if (MULTI) s[x][2 * y] = p0, s[x][2 * y + 1] = p1;
        }
      }
      if (MULTI && !whole) {
        // A value that is not finite must not reach the queries that do not see its slot
        // (0 * NaN): the product takes zeros in such places, and what the queries that see
        // them get is added here.
        uint32_t bad = 0;
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int u = 0; u < DC; ++u)
            bad |= Mma<T>::not_finite(vf[x][u].x) | Mma<T>::not_finite(vf[x][u].y) |
                   Mma<T>::not_finite(vf[x][u].z) | Mma<T>::not_finite(vf[x][u].w);
        if (__any_sync(0xffffffffu, bad != 0)) {
          for (int e = 0; e < TK; ++e) {
            const int from = (lane & 28) | (e >> 1 & 3), j = j0 + e;
            float w[2];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const float lo = e & 1 ? s[0][2 * y + 1] : s[0][2 * y], hi = e & 1 ? s[1][2 * y + 1] : s[1][2 * y];
              w[y] = __shfl_sync(0xffffffffu, e < 8 ? lo : hi, from);
            }
            if (j >= jend) break;
#pragma unroll
            for (int u = 0; u < DC; ++u)
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const int d = 64 * u + 16 * t + 8 * x;
                float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                if (FULL || d < D) load8(vb + j * a.kv_slot + d, v);
#pragma unroll
                for (int k = 0; k < 8; ++k)
#pragma unroll
                  for (int y = 0; y < 2; ++y)
                    if (w[y] != 0.f && !isfinite(v[k]))
                      o[8 * u + k][2 * y + x] = fmaf(w[y], v[k], o[8 * u + k][2 * y + x]);
              }
          }
#pragma unroll
          for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int u = 0; u < DC; ++u) {
              vf[x][u].x = Mma<T>::finite(vf[x][u].x);
              vf[x][u].y = Mma<T>::finite(vf[x][u].y);
              vf[x][u].z = Mma<T>::finite(vf[x][u].z);
              vf[x][u].w = Mma<T>::finite(vf[x][u].w);
            }
        }
      }
#pragma unroll
      for (int u = 0; u < DC; ++u) {
        const uint32_t* v0 = reinterpret_cast<const uint32_t*>(&vf[0][u]);
        const uint32_t* v1 = reinterpret_cast<const uint32_t*>(&vf[1][u]);
        const uint32_t* v2 = reinterpret_cast<const uint32_t*>(&vf[2][u]);
        const uint32_t* v3 = reinterpret_cast<const uint32_t*>(&vf[3][u]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          Mma<T>::run(o[8 * u + 2 * w], w16[0], w16[1], w16[2], w16[3], __byte_perm(v0[w], v1[w], 0x5410),
                      __byte_perm(v2[w], v3[w], 0x5410));
          Mma<T>::run(o[8 * u + 2 * w + 1], w16[0], w16[1], w16[2], w16[3], __byte_perm(v0[w], v1[w], 0x7632),
                      __byte_perm(v2[w], v3[w], 0x7632));
        }
      }
      }
      load_v();
      if (!again) break;
    }

    // The warps' results into shared memory.
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      l[y] += __shfl_xor_sync(0xffffffffu, l[y], 1);
      l[y] += __shfl_xor_sync(0xffffffffu, l[y], 2);
      const int m = g + 8 * y;
      if (m >= nG) continue;
      if (t == 0) warp_ml[warp][m] = make_float2(ref[y], l[y]);
#pragma unroll
      for (int u = 0; u < DC; ++u)
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const int j = 8 * u + 4 * w;
            *vec_at(warp, m, 16 * u + 4 * t + 2 * x + w) =
                make_float4(o[j][2 * y + x], o[j + 1][2 * y + x], o[j + 2][2 * y + x], o[j + 3][2 * y + x]);
          }
    }
    if (more_units) load_q(next);
    // A unit of this block alone is finished here, the prefix's parts joined with the warps'.
    const bool alone = p.first >= c0 && p.end <= c1;
    const int extra = alone ? a.p_splits : 0, slot = 2 * c + (p.first >= c0);
    const int64_t row0 = prefix_index(a, p.r, p.h, 0);
    if (extra) {
      wait_before();  // the prefix's kernel may have run beside this one
      for (int x = tid; x < extra * 16; x += NT)
        if ((x & 15) < nG) part_ml[x >> 4][x & 15] = __ldcg(a.prefix_ml + (int64_t)(x >> 4) * all_rows + row0 + (x & 15));
    }
    __syncthreads();
    if (tid < nG) {
      float M = -INFINITY;
#pragma unroll
      for (int k = 0; k < NW; ++k) M = fmaxf(M, warp_ml[k][tid].x);
      for (int k = 0; k < extra; ++k) M = fmaxf(M, part_ml[k][tid].x);
      const float at = M == -INFINITY ? 0.f : M;
      float L = 0.f;
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        const float f = ex2(warp_ml[k][tid].x - at);
        factor[k][tid] = f;
        L = fmaf(warp_ml[k][tid].y, f, L);
      }
      for (int k = 0; k < extra; ++k) {
        const float f = part_ml[k][tid].y == 0.f ? 0.f : ex2(part_ml[k][tid].x - at);
        factor[NW + k][tid] = f;
        L = fmaf(part_ml[k][tid].y, f, L);
      }
      joined[tid] = make_float2(M, L);
    }
    __syncthreads();
    {
      // This thread's vectors of four side by side: their loads are in flight together.
      constexpr int ITEMS = (16 * DC * 16 + NT - 1) / NT;
      int m[ITEMS], d[ITEMS];
      float4 v[ITEMS];
#pragma unroll
      for (int x = 0; x < ITEMS; ++x) v[x] = make_float4(0.f, 0.f, 0.f, 0.f);
      auto add = [&](int x, float4 y, float f) {
        v[x].x = fmaf(y.x, f, v[x].x);
        v[x].y = fmaf(y.y, f, v[x].y);
        v[x].z = fmaf(y.z, f, v[x].z);
        v[x].w = fmaf(y.w, f, v[x].w);
      };
#pragma unroll
      for (int x = 0; x < ITEMS; ++x) {
        m[x] = (tid + x * NT) / row_vecs;
        d[x] = (tid + x * NT - m[x] * row_vecs) * 4;
        if (m[x] < nG) {
#pragma unroll
          for (int k = 0; k < NW; ++k) add(x, *vec_at(k, m[x], d[x] >> 2), factor[k][m[x]]);
        }
      }
#pragma unroll 4
      for (int k = 0; k < extra; ++k)
#pragma unroll
        for (int x = 0; x < ITEMS; ++x)
          if (m[x] < nG)
            add(x, __ldcg(reinterpret_cast<const float4*>(a.prefix_o + ((int64_t)k * all_rows + row0 + m[x]) * D + d[x])),
                factor[NW + k][m[x]]);
#pragma unroll
      for (int x = 0; x < ITEMS; ++x) {
        if (m[x] >= nG) continue;
        if (alone)
          write_out(p, m[x], d[x], v[x], joined[m[x]].y);
        else
          *reinterpret_cast<float4*>(a.part_o + ((int64_t)slot * 16 + m[x]) * D + d[x]) = v[x];
      }
    }
    if (tid < nG) {
      if (alone)
        write_lse(p, tid);
      else
        a.part_ml[slot * 16 + tid] = joined[tid];
    }
    if (!alone) shared_part[shared_parts++] = p;
    if (a.status && tid == 0 && p.h == K - 1 && p.end <= c1) {
      const int e = a.lengths ? a.lengths[p.r] : a.capacity, s = a.starts ? a.starts[p.r] : 0;
      a.status[p.r] = (e < 0 || e > a.capacity || s < 0 || s > max(e, 0)) ? 8 : 0;
    }
    __syncthreads();
    if (!more_units) break;
    p = next;
  }

  // The block that arrives last at a unit (past kMaxFlat parts: at its group of parts,
  // then at the unit) joins; both units' arrivals go out together.
  auto arrives_last = [&](unsigned* counter, int count) {
    const bool is_last = arrive(counter) == (unsigned)count - 1u;
    if (is_last) *counter = 0u;
    return is_last;
  };
  __syncthreads();
  if (tid < shared_parts) {
    const Part& p = shared_part[tid];
    const int c_first = block_of(p.first), parts = block_of(p.end - 1) - c_first + 1;
    const int first = c_first + (c - c_first) / kJoin * kJoin;
    sh_last[tid] = parts > kMaxFlat ? arrives_last(a.counters + (int64_t)a.rows * K + 2 * first + (first == c_first),
                                                   min(kJoin, c_first + parts - first))
                                    : arrives_last(a.counters + p.r * K + p.h, parts);
  }
  __syncthreads();
  for (int x = 0; x < shared_parts; ++x) {
    if (!sh_last[x]) continue;
    const Part p = shared_part[x];
    const int c_first = block_of(p.first), parts = block_of(p.end - 1) - c_first + 1;
    int step = 1, count = parts;
    if (parts > kMaxFlat) {
      const int first = c_first + (c - c_first) / kJoin * kJoin;
      join(p, c_first, first, 1, min(kJoin, c_first + parts - first), false, std::false_type());
      step = kJoin;
      count = (parts + kJoin - 1) / kJoin;
      __syncthreads();
      if (tid == 0) sh_last[x] = arrives_last(a.counters + p.r * K + p.h, count);
      __syncthreads();
      if (!sh_last[x]) continue;
    }
    join(p, c_first, c_first, step, count, true, std::true_type());
  }
  wait_before();
}

// Accumulated weights from the scores that the token kernel left: one thread per slot.
__global__ void __launch_bounds__(256) scores_weights_kernel(const __grid_constant__ AttnArgs a) {
  const int unit = blockIdx.y, h = unit % a.kv_heads, r = unit / a.kv_heads;
  const RowSpan sp = row_span(a, r);
  const int j = blockIdx.x * 256 + threadIdx.x;
  wait_before();
  if (j >= sp.end || j < sp.start) return;
  const int nG = a.n * a.group;
  const float* s = a.scores + (int64_t)unit * nG * a.capacity + j;
  const float* lse = a.lse + (int64_t)unit * nG;
  float sum = 0.f;
  for (int i = 0; i < a.n; ++i) {
    const int p = sp.end - a.n + i;
    if (!slot_seen(a, sp.start, p, window_low(a, sp.start, p), j)) continue;
    for (int g = 0; g < a.group; ++g) {
      const int m = i * a.group + g;
      sum += ex2(s[(int64_t)m * a.capacity] - lse[m]);
    }
  }
  a.weights[r * a.w_row + h * a.w_head + j] += sum;
}

// Accumulated weights of calls with many query rows: w[slot] += sum of 2^(s - lse) over
// the group's rows.  A warp holds 16 slots' keys as the A operand and walks the query
// rows 8 at a time as the B operand, both straight from global memory as above; the
// queries come from L1 for seven of a block's eight warps.  One warp owns its slots, so
// the sum's order is fixed and no atomics are needed.  Bound by the products.
// LOW: the keys of a 4-bit cache in two pieces of T.
template <typename T, int DC, bool FULL, bool LOW>
__global__ void __launch_bounds__(NT) attn_weights16_kernel(const __grid_constant__ AttnArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int unit = blockIdx.y, h = unit % a.kv_heads, r = unit / a.kv_heads, nG = a.n * a.group, vecs = a.dim >> 3;
  const RowSpan sp = row_span(a, r);
  const int j0 = (blockIdx.x * NW + warp) * 16;
  if (j0 >= sp.end || j0 + 16 <= sp.start) return;
  uint4 kf[2][2 * DC], kl[2][2 * DC], qf[2 * DC], qn[2 * DC];
  auto load_k = [&](uint4(&to)[2][2 * DC], const void* from) {
    const T* kb = static_cast<const T*>(from) + r * a.kv_row + h * a.kv_head;
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int u = 0; u < 2 * DC; ++u)
        to[x][u] = load_stream(kb + (j0 + g + 8 * x) * a.kv_slot + (4 * u + t) * 8,
                               j0 + g + 8 * x < sp.end && (FULL || 4 * u + t < vecs));
  };
  load_k(kf, LOW ? a.w_k : a.k);
  if (LOW) load_k(kl, a.w_low);
  const int first_pos = sp.end - a.n;
  int m_first, m_end;
  weight_rows(a, sp, j0, 16, blockIdx.z, m_first, m_end);
  // Past the last row that row again, with a sum of infinity: its exponentials are zero, and NaN only
  // where the row's own is (of a zero query and an infinite key they would be anyway).
  const int m_last = max(m_end - 1, 0);
  auto load_q = [&](int m0) {
    const int m = min(m0 + g, m_last), i = m / a.group;
    const T* src = static_cast<const T*>(a.q) + r * a.q_row + i * a.q_tok +
                   (int64_t)(h * a.group + m - i * a.group) * a.q_head;
#pragma unroll
    for (int u = 0; u < 2 * DC; ++u)
      qn[u] = FULL || 4 * u + t < vecs ? __ldg(reinterpret_cast<const uint4*>(src) + 4 * u + t)
                                       : make_uint4(0u, 0u, 0u, 0u);
  };
  float sum[2] = {0.f, 0.f};
  const float* lse = a.lse + (int64_t)unit * nG;
  load_q(m_first);
  for (int m0 = m_first; m0 < m_end; m0 += 8) {
#pragma unroll
    for (int u = 0; u < 2 * DC; ++u) qf[u] = qn[u];
    load_q(m0 + 8);
    float l[2], c[2][4];
    int pos[2], low[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int m = m0 + 2 * t + e;
      l[e] = m < m_end ? lse[m] : INFINITY;
      pos[e] = first_pos + min(m, m_last) / a.group;
      low[e] = window_low(a, sp.start, pos[e]);
#pragma unroll
      for (int k = 0; k < 4; ++k) c[e][k] = 0.f;
    }
#pragma unroll
    for (int u = 0; u < 2 * DC; ++u) {
      Mma<T>::run(c[0], kf[0][u].x, kf[1][u].x, kf[0][u].y, kf[1][u].y, qf[u].x, qf[u].y);
      Mma<T>::run(c[1], kf[0][u].z, kf[1][u].z, kf[0][u].w, kf[1][u].w, qf[u].z, qf[u].w);
      if (LOW) {
        Mma<T>::run(c[0], kl[0][u].x, kl[1][u].x, kl[0][u].y, kl[1][u].y, qf[u].x, qf[u].y);
        Mma<T>::run(c[1], kl[0][u].z, kl[1][u].z, kl[0][u].w, kl[1][u].w, qf[u].z, qf[u].w);
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int j = j0 + g + 8 * (k >> 1), e = k & 1;
      if (slot_seen(a, sp.start, pos[e], low[e], j)) sum[k >> 1] += ex2((c[0][k] + c[1][k]) * a.scale - l[e]);
    }
  }
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], 1);
    sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], 2);
    const int j = j0 + g + 8 * x;
    if (t == 0 && j >= sp.start && j < sp.end) add_weight(a, unit, r, h, j, blockIdx.z, sum[x]);
  }
}

template <typename T, int DC, bool FULL, bool MULTI>
cudaError_t token(const AttnArgs& a, int blocks, cudaStream_t stream) {
  constexpr size_t smem = sizeof(float) * NW * 16 * DC * 64;
  const cudaError_t e = allow_smem<attn_token_kernel<T, DC, FULL, MULTI>>(smem);
  if (e != cudaSuccess) return e;
  // Beside the prefix's kernel where that leaves SMs: its results are needed at the joins only.
  return launch_after(a.prefix != 0, attn_token_kernel<T, DC, FULL, MULTI>, dim3(blocks), NT, smem, stream, a, blocks);
}

// (The forms for 72 to 120 dimensions spill 20 to 52 bytes at 255 registers.)
template <typename T, bool MULTI> cudaError_t token_dim(const AttnArgs& a, int blocks, cudaStream_t stream) {
  if (a.dim == 128) return token<T, 2, true, MULTI>(a, blocks, stream);
  if (a.dim == 64) return token<T, 1, true, MULTI>(a, blocks, stream);
  return a.dim < 64 ? token<T, 1, false, MULTI>(a, blocks, stream) : token<T, 2, false, MULTI>(a, blocks, stream);
}

template <typename T> cudaError_t token_any(const AttnArgs& a, int blocks, cudaStream_t stream) {
  return a.n > 1 ? token_dim<T, true>(a, blocks, stream) : token_dim<T, false>(a, blocks, stream);
}

}  // namespace

cudaError_t launch_attn_token(const AttnArgs& a, int blocks, cudaStream_t stream) {
  return a.dtype == 1 ? token_any<__half>(a, blocks, stream) : token_any<__nv_bfloat16>(a, blocks, stream);
}

template <typename T, bool LOW> cudaError_t weights16(const AttnArgs& a, cudaStream_t stream) {
  const dim3 grid((unsigned)((a.capacity + NW * 16 - 1) / (NW * 16)), (unsigned)(a.rows * a.kv_heads),
                  (unsigned)a.w_splits);
  if (a.dim == 128)
    attn_weights16_kernel<T, 2, true, LOW><<<grid, NT, 0, stream>>>(a);
  else if (a.dim > 64)
    attn_weights16_kernel<T, 2, false, LOW><<<grid, NT, 0, stream>>>(a);
  else
    attn_weights16_kernel<T, 1, false, LOW><<<grid, NT, 0, stream>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_weights16(const AttnArgs& a, cudaStream_t stream) {
  if (a.w_low) return a.dtype == 1 ? weights16<__half, true>(a, stream) : weights16<__nv_bfloat16, true>(a, stream);
  return a.dtype == 1 ? weights16<__half, false>(a, stream) : weights16<__nv_bfloat16, false>(a, stream);
}

cudaError_t launch_scores_weights(const AttnArgs& a, cudaStream_t stream) {
  return launch_after(true, scores_weights_kernel,
                      dim3((unsigned)((a.capacity + 255) / 256), (unsigned)(a.rows * a.kv_heads)), 256, 0, stream, a);
}

}  // namespace sv
