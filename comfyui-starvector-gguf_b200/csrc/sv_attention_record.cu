// sv_attention_record.cu -- attention of few query rows per key/value head over the
// cache held in 4 bits (sv_record.cuh): single tokens and drafts.  A unit's records are read once; rows
// past 16 of a head (float32: 8) are units of their own, up to four, each of which reads them again.
//
// Mathematics.  Row m of a unit (cache row r, key/value head h, 8 or 16 of its query rows):
// with a key's groups k_d = mid_g + scale_g (c_d - 8),
//   q . k = sum_g scale_g (sum_{d in g} q_d c_d - 8 sum_{d in g} q_d) + sum_g mid_g sum_{d in g} q_d.
// The codes are whole numbers below 16, which float16 holds exactly: a nibble masked out
// of a word is, read as float16, its subnormal c 2^-24 (or, four bits further up, c 2^-20:
// those dimensions' queries are divided by 16), so a key needs no arithmetic before the
// tensor core takes it.  The queries are brought into float16's upper range by a power of two
// per row, which loses nothing of a bfloat16.  The scales multiply the groups' sums in f32; the rest,
// sum_g (mid_g - 8 scale_g) times the queries' group sums, is one product more, whose A operand is the
// record's pairs as they lie (the group sums in two halves, 22 bits).  So scores are as exact as those of f32 keys.
// Values are formed in float16, v = scale (c - 8) + mid rounded once, and the weights rounded to
// float16, for float16 outputs in two halves: one such rounding is about what the output's own adds (error of
// one token's output 0.0003 against 64 bits, 0.0002 that of the output's rounding alone; with both 0.00032).
// Float32: queries in two float16 pieces, weights and values in three bfloat16 pieces each and the six products
// that count.
// The softmax as in sv_attention_token.cu: the reference moves only when a score exceeds it by
// 2^8.  Weights are held to 2^-32 of the heaviest (kRaised).
//
// Both products are turned round, S^T = K Q^T and O^T = V^T P^T (mma.m16n8k16): slots and
// dimensions fill the 16 rows, and the query rows take columns in eights, so that four heads of
// a group do not pay for sixteen; weights pass from the one to the other by a transposition
// (movmatrix).
//
// What bounds it: the instructions that turn codes into operands, and the products.  128 dimensions, cycles of a
// scheduler per 16 slots (the memory's rate allows 450): 532 with four query rows (5.4 TB/s of
// records), 727 with nine, of which about 300 are the products' and 300 the integer instructions'.  64 rows of 36/4
// heads over 4096 slots take 66 us (2.6 TB/s; floor 26 us), 8 rows over up to 16384 slots 29 us (floor 9.6), of
// which start, units' ends and joins are a large part.
// A warp takes tiles of 16 or 32 slots through a ring in shared memory of its own (cp.async, zeros for slots past
// the end): registers alone would keep too few bytes in flight, since 16 slots are only 2560.  Rows of a tile are taken in an order in which neither the keys' nor the
// values' reads meet in a bank (slot_at).
//
// Work split and joins as in sv_attention_token.cu: one list of chunks (a tile per warp) over all
// units, cut into equal parts, one per block; the last block to arrive joins a unit that
// several share, in block order.
#include <climits>
#include <type_traits>

#include "sv_attention.h"
#include "sv_record.cuh"

namespace sv {
namespace {

constexpr int kJoin = 16;      // parts per first-level group
constexpr int kMaxFlat = 32;   // parts joined in one level
constexpr float kSlack = 8.f;  // log2 by which a score may exceed its reference
// 16-bit calls: log2 of the weight that a new reference stands for, so that weights use float16's range up to 2^15 and
// those down to 2^-32 of the reference do not vanish in it (with a reference of weight 1 a slot that outweighed 16384
// others by 2^24.5 each lost or gained two fifths of their share).
constexpr float kRaised = 7.f;
constexpr float kNever = -0x1.fp127f;  // a reference before the first score

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// d = a b; d += a b.
__device__ __forceinline__ void mma_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_add(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Two values rounded to bfloat16, which are taken off them.
__device__ __forceinline__ uint32_t next_piece(float2& x) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x.x, x.y);
  const float2 f = __bfloat1622float2(h);
  x.x -= f.x;
  x.y -= f.y;
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Float32: the values of nibble j of two slots' 16-bit halves, in three bfloat16 pieces each.
__device__ __forceinline__ void pieces(uint32_t w, int j, uint32_t scale, uint32_t mid, uint32_t& a, uint32_t& b, uint32_t& c) {
  const float2 s = __half22float2(*reinterpret_cast<const __half2*>(&scale)), m = __half22float2(*reinterpret_cast<const __half2*>(&mid));
  const float c0 = __uint_as_float((w >> 4 * j & 15u) | 0x4b000000u) - 8388616.f;  // 2^23 + c - (2^23 + 8)
  const float c1 = __uint_as_float((w >> (16 + 4 * j) & 15u) | 0x4b000000u) - 8388616.f;
  float2 v = make_float2(fmaf(s.x, c0, m.x), fmaf(s.y, c1, m.y));
  a = next_piece(v);
  b = next_piece(v);
  c = next_piece(v);
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
// (a & b) | c as one instruction: b and c in registers whose values the compiler does not see (as
// immediates they would take an instruction each).
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t hidden(uint32_t x) {
  uint32_t y;
  asm volatile("mov.u32 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy16_or_zeros(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint32_t load1(uint32_t at) {
  uint32_t x;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(at));
  return x;
}
template <int N> __device__ __forceinline__ void load2(uint32_t (&x)[N], uint32_t at) {
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(x[0]), "=r"(x[1]) : "r"(at));
}
__device__ __forceinline__ void load4(uint32_t (&x)[4], uint32_t at) {
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(at));
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
template <int NI, int SUB> struct Form {
  static constexpr int TK = 16 * SUB;                         // slots of a tile
  static constexpr int REC = 16 * NI + 16;                    // bytes
  static constexpr int NG = NI > 2 ? NI : 2 * NI;             // groups
  static constexpr int NB = NI > 2 ? 2 : 1;                   // words of a value that one thread turns into operands
  static constexpr int TILE = TK * REC;                       // bytes of a tile's keys (or values)
};


// Like sv_attention_token.cu's: [a0, a1) the sinks before the window, [b0, b1) the rest.
struct RowTiles {
  int start, end, a0, a1, b0, b1, ta, tiles;
};

template <int TK> __device__ __noinline__ RowTiles row_tiles(const AttnArgs& a, int r) {
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

// Empty places of the list behind every unit's chunks, where blocks take eight and more: what beginning and ending a
// unit costs, so that blocks of many units get fewer chunks (64 rows over 4096 slots 64 us, 66 without, when they came in: some blocks
// worked 8 us longer).
constexpr int kBetween = 2;

// A place in the list of chunks: chunk k of unit (r, h), h counting the heads' groups of rows.
template <int NW, int TK> struct Place {
  int r, h, k, chunks;
  RowTiles rt;
  __device__ __forceinline__ void row(const AttnArgs& a, int r_) {
    r = r_;
    rt = row_tiles<TK>(a, r_);
    chunks = (rt.tiles + NW - 1) / NW;
  }
};

// NI blocks of 32 dimensions, NT column tiles of eight query rows, NW warps, rings of RING tiles.
// MULTI: more than one query per row.
// A tile is SUB times 16 slots, whose steps have nothing to wait for from one another.
template <typename T, int NI, int NT, int SUB, int NW, int RING, bool MULTI>
__global__ void __launch_bounds__(NW * 32, 1)
    attn_record_kernel(const __grid_constant__ AttnArgs a, const int blocks_max, const int row_groups) {
  using F = Form<NI, SUB>;
  constexpr int TK = F::TK, REC = F::REC, NG = F::NG, NB = F::NB, MT = 4 * NB, ROWS = 8 * NT, THREADS = NW * 32;
  constexpr int OS = 32 * NI;  // dimensions of the warps' outputs
  constexpr bool HALVES = std::is_same<T, __half>::value, FULL = std::is_same<T, float>::value;
  constexpr int QP = FULL ? 2 : 1, WP = FULL ? 3 : HALVES ? 2 : 1;  // pieces of a query, of a weight
  constexpr bool KEEP_Q = NT * NW <= 16 && !FULL;                   // the queries' operands in registers
  constexpr uint32_t kOnes = 0x3c003c00u;
  constexpr float kRaise = FULL ? 0.f : kRaised, kMove = kSlack + kRaise;
  // [NW][RING][keys, values of a tile], then [NW][ROWS][OS] floats.
  extern __shared__ __align__(16) unsigned char ring_bytes[];
  float* const outs = reinterpret_cast<float*>(ring_bytes + NW * RING * 2 * F::TILE);
  __shared__ float warp_m[NW][ROWS], warp_l[NW][ROWS];
  __shared__ float factor[kMaxFlat > NW ? kMaxFlat : NW][ROWS];
  __shared__ float2 part_ml[kMaxFlat][ROWS];
  __shared__ float2 joined[ROWS];
  __shared__ uint4 sh_q[QP][NT][NI][32];
  __shared__ uint2 sh_qm[NT][32];
  __shared__ float sh_fr[ROWS];
  __shared__ int scan[NW];
  __shared__ int sh_row, sh_before, sh_last[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int group = a.group, nG = MULTI ? a.n * group : group, K = a.kv_heads * row_groups, D = a.dim;

  // The warps' outputs: 4 dimensions c of row m, placed so that the fragments' writes do not meet in a bank.
  auto vec_at = [&](int w, int m, int c) {
    return reinterpret_cast<float4*>(outs) + (w * ROWS + m) * (OS / 4) + (c ^ (m >> 1 & 3) ^ (OS >= 128 ? c >> 2 & 4 : 0));
  };

  // (Launched while the kernel before it ends; the next one may be, too.)
  wait_before();
  launch_dependents();

  // Chunks of all rows, every head of a row having as many: see sv_attention_token.cu.
  const int per = (a.rows + THREADS - 1) / THREADS, row0 = tid * per;
  int mine = 0;
  for (int x = row0; x < min(row0 + per, a.rows); ++x) mine += (row_tiles<TK>(a, x).tiles + NW - 1) / NW;
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
  const int between = total * K >= 8 * blocks_max ? kBetween : 0;
  mine += between * max(min(per, a.rows - row0), 0);
  upto += between * min(row0 + per, a.rows);
  total += between * a.rows;
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
      const int chunks = (row_tiles<TK>(a, x).tiles + NW - 1) / NW + between;
      if (c0 < (at + chunks) * K) break;
      at += chunks;
    }
    sh_row = x;
    sh_before = at;
  }
  __syncthreads();
  Place<NW, TK> p;
  p.row(a, sh_row);
  {
    const int off = c0 - sh_before * K;
    p.h = off / (p.chunks + between);
    p.k = off - p.h * (p.chunks + between);
  }
  int before = sh_before;  // places (of one head) before row p.r
  int f_place = c0;        // the next chunk to fetch
  if (p.k >= p.chunks) {   // behind a unit's chunks: on to the next one, if it begins here
    f_place += p.chunks + between - p.k;
    if (f_place >= c1) return;
    p.k = 0;
    if (++p.h == K) {
      p.h = 0;
      before += p.chunks + between;
      p.row(a, p.r + 1);
    }
  }

  // ---- copies: this warp's tile of chunk f, the f-th place ahead.  The next `runs` of them are whole
  // tiles of one unit, each a run of bytes f_step behind the one before.
  Place<NW, TK> f = p;
  int runs = 0;
  const unsigned char *f_k, *f_v;
  const int64_t f_step = (int64_t)NW * TK * a.kv_slot;
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(ring_bytes) + warp * RING * 2 * F::TILE;
  uint32_t put = ring + lane * 16;
  // The place f by slots (the end of a unit, sinks, other strides), or none; then what comes after it.
  auto fetch_slots = [&]() {
    if (f_place >= c1) return;
    const int tile = f.k * NW + warp;
    const int64_t base = f.r * a.kv_row + (f.h / row_groups) * a.kv_head;
    if (tile < f.rt.tiles) {
      const bool in_a = tile < f.rt.ta;
      const int j0 = in_a ? f.rt.a0 + tile * TK : f.rt.b0 + (tile - f.rt.ta) * TK;
      const int count = min(TK, (in_a ? f.rt.a1 : f.rt.b1) - j0);
#pragma unroll 1
      for (int x = lane; x < 2 * F::TILE / 16; x += 32) {
        const int in = x >= F::TILE / 16 ? x - F::TILE / 16 : x, slot = in / (REC / 16);
        const int64_t at = base + (j0 + slot) * a.kv_slot + (in - slot * (REC / 16)) * 16;
        copy16_or_zeros(put + (x - lane) * 16, static_cast<const unsigned char*>(x == in ? a.k : a.v) + (slot < count ? at : 0),
                        slot < count);
      }
    }
    ++f_place;
    if (++f.k == f.chunks) {
      f.k = 0;
      f_place += between;
      if (++f.h == K) {
        f.h = 0;
        if (f.r + 1 < a.rows) f.row(a, f.r + 1);  // (past the last chunk of all nothing is looked at)
      }
    }
  };
  auto find_runs = [&]() {
    runs = 0;
    const int tile = f.k * NW + warp, f_hi = f.rt.ta + (f.rt.b1 - f.rt.b0) / TK;
    if (f_place >= c1 || a.kv_slot != REC || tile < f.rt.ta || tile >= f_hi) return;
    // Not a unit's last chunk, after which the place moves on.
    runs = min(min((f_hi - tile + NW - 1) / NW, f.chunks - 1 - f.k), c1 - f_place);
    const int64_t at = f.r * a.kv_row + (f.h / row_groups) * a.kv_head + (f.rt.b0 + (tile - f.rt.ta) * TK) * a.kv_slot;
    f_k = static_cast<const unsigned char*>(a.k) + at + lane * 16;
    f_v = static_cast<const unsigned char*>(a.v) + at + lane * 16 - F::TILE;
    f.k += runs;
    f_place += runs;
  };
  find_runs();
  auto fetch = [&]() {
    if (runs > 0) {
#pragma unroll
      for (int x = 0; x < 2 * F::TILE / 512; ++x) {
        constexpr int K = F::TILE / 16;  // copies of keys
        copy16(put + x * 512, (32 * x + 32 <= K || (32 * x < K && lane + 32 * x < K) ? f_k : f_v) + x * 512);
      }
      --runs;
      f_k += f_step;
      f_v += f_step;
    } else {
      fetch_slots();
      find_runs();
    }
    put = put + 2 * F::TILE == ring + lane * 16 + RING * 2 * F::TILE ? ring + lane * 16 : put + 2 * F::TILE;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  // ---- queries, for the whole block, row tile u by warp u: the B operand of each step over 16 dimensions, the
  // groups' sums in halves, the rows' factors
  using Four = std::conditional_t<FULL, uint4, uint2>;  // four values as they lie
  Four raw[NI][2];
  auto load_q = [&](int r, int h) {
    const int head = h / row_groups, m = (h - head * row_groups) * ROWS + 8 * warp + g, i = MULTI ? m / group : 0;
    const T* src = static_cast<const T*>(a.q) + r * a.q_row + i * a.q_tok + (int64_t)(head * group + m - i * group) * a.q_head;
#pragma unroll
    for (int b = 0; b < NI; ++b)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int d = 32 * b + 16 * e + 4 * t;
        raw[b][e] = Four();
        if (warp < NT && m < nG && d < D) raw[b][e] = __ldg(reinterpret_cast<const Four*>(src + d));
      }
  };
  auto make_q = [&]() {
    if (warp >= NT) return;
    float x[NI][2][4], most = 0.f;
#pragma unroll
    for (int b = 0; b < NI; ++b)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const T* y = reinterpret_cast<const T*>(&raw[b][e]);
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
    for (int b = 0; b < NI; ++b) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          x[b][e][k] *= up;
          sum[NI > 2 ? b : 2 * b + e] += x[b][e][k];
        }
#pragma unroll
      for (int y = 0; y < QP; ++y) {
        const uint4 q = make_uint4(pack16(x[b][0][0], x[b][0][1]), pack16(x[b][0][2] * 0.0625f, x[b][0][3] * 0.0625f),
                                   pack16(x[b][1][0], x[b][1][1]), pack16(x[b][1][2] * 0.0625f, x[b][1][3] * 0.0625f));
        sh_q[y][warp][b][lane] = q;
        if (y + 1 < QP) {  // what the rounding left
          const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
            x[b][k >> 1][2 * (k & 1)] -= k & 1 ? 16.f * h.x : h.x;
            x[b][k >> 1][2 * (k & 1) + 1] -= k & 1 ? 16.f * h.y : h.y;
          }
        }
      }
    }
    // Group t's sum, 2^10 above the keys' units (in theirs the halves would be float16's subnormals: scores off by 2^-15 of
    // the largest query times the middles); in halves, for scale (times -8) and mid.
    float own = 0.f;
#pragma unroll
    for (int k = 0; k < NG; ++k) {
      sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 1);
      sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 2);
      if (k == t) own = sum[k] * 0x1p-14f;
    }
    const float high = __half2float(__float2half_rn(own));
    sh_qm[warp][lane] = make_uint2(pack16(-8.f * high, high), pack16(-8.f * (own - high), own - high));
    // |scale| 2^(ex - 141 + 24).  (Past 2^112 a smaller factor: it keeps scores past f32's range within it, and any two
    // that differ are 2^40 apart by then.  A factor of zero would make NaN of hidden slots' -infinity.)
    if (t == 0) {
      const float factor = fabsf(a.scale) * __uint_as_float((uint32_t)min(ex, 254) << 23) * 1024.f;
      sh_fr[8 * warp + g] = fminf(fmaxf(factor, 0x1p-126f), 0x1p112f);
    }
  };

  auto write_out = [&](int r, int head, int m, int d, float4 x, float L) {  // m: row of the head's nG
    if (d >= D) return;
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const int i = MULTI ? m / group : 0;
    T* out = static_cast<T*>(a.out) + (((int64_t)r * a.n + i) * a.heads + head * group + m - i * group) * D + d;
    alignas(16) T y[4] = {from_float<T>(x.x * inv), from_float<T>(x.y * inv), from_float<T>(x.z * inv), from_float<T>(x.w * inv)};
    *reinterpret_cast<Four*>(out) = *reinterpret_cast<const Four*>(y);
  };
  auto write_lse = [&](int r, int head, int m, float2 j) {
    if (a.lse) a.lse[(int64_t)(r * a.kv_heads + head) * nG + m] = j.y == 0.f ? INFINITY : j.x + log2f(j.y);
  };

  // The units this block shares with others: the one it starts in and the one it ends in at most.
  struct Shared { int r, h, first, end; };
  Shared shared_part[2];
  int shared_parts = 0;
  constexpr int VECS = ROWS * (OS / 4), ITEMS = (VECS + THREADS - 1) / THREADS;

  auto arrives_last = [&](unsigned* counter, int count) {
    const bool is_last = arrive(counter) == (unsigned)count - 1u;
    if (is_last) *counter = 0u;
    return is_last;
  };
  // By one thread, once the part's results are written: whether the others' are all there (past kMaxFlat parts:
  // of its group of parts).
  auto arrive_at = [&](const Shared& q) {
    const int c_first = block_of(q.first), parts = block_of(q.end - 1) - c_first + 1;
    const int b0 = c_first + (c - c_first) / kJoin * kJoin;
    return parts > kMaxFlat ? arrives_last(a.counters + (int64_t)a.rows * K + 2 * b0 + (b0 == c_first), min(kJoin, c_first + parts - b0))
                            : arrives_last(a.counters + q.r * K + q.h, parts);
  };
  load_q(p.r, p.h);  // (behind the tiles' loads they would wait for them)
#pragma unroll 1
  for (int k = 0; k < RING - 1; ++k) fetch();
  uint32_t get = ring;
  const uint32_t k_even = hidden(0x000f000fu), k_odd = hidden(0x00f000f0u), k_1024 = hidden(0x64006400u), k_64 = hidden(0x54005400u);
  bool last_shared = false;  // whether the part before was
  make_q();
  __syncthreads();
  for (;;) {  // units
    const int head = p.h / row_groups, m0 = (p.h - head * row_groups) * ROWS, rows_here = min(ROWS, nG - m0);
    const int first = before * K + p.h * (p.chunks + between), end = first + p.chunks, stop = min(end, c1);
    const bool more = end + between < c1;  // the next unit begins here, too
    const int at = max(c0, first);
    const RowTiles rt = p.rt;
    const int pos_first = rt.end - a.n, low_last = window_low(a, rt.start, rt.end - 1);
    // This warp's tiles of the part; in [w_lo, w_hi) every row sees the whole tile.
    const int chunks = stop - at, tile0 = (at - first) * NW + warp;
    const int valid = min(chunks, max(0, (rt.tiles - tile0 + NW - 1) / NW));
    const int w_lo = rt.ta + (MULTI ? (low_last - rt.b0 + TK - 1) / TK : 0);
    const int w_hi = rt.ta + ((MULTI ? min(rt.b1, pos_first + 1) : rt.b1) - rt.b0) / TK;
    // As numbers of the loop's rounds.
    const int k_lo = (w_lo - tile0 + NW - 1) / NW, k_hi = w_hi > tile0 ? (w_hi - tile0 + NW - 1) / NW : 0;
    const int s0 = slot_at(g), s1 = slot_at(g + 8);
    const uint32_t va = slot_at(2 * t) * REC, vb = slot_at(2 * t + 1) * REC;  // rows 8..15: the slots behind them
    float fr[NT][2], from[NT][2];  // from: a row's reference, negative (far below any score before the first)
    float o[NT][MT][4], l[NT][2];
    bool huge = false;  // a reference past 2^20, where the fused product's exactness would set its own maximum far off
    uint4 qb[KEEP_Q ? NT : 1][NI];
    uint2 qm[NT];
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      if constexpr (KEEP_Q) {
        qm[u] = sh_qm[u][lane];
#pragma unroll
        for (int b = 0; b < NI; ++b) qb[u][b] = sh_q[0][u][b][lane];
      }
      const float2 both = *reinterpret_cast<const float2*>(&sh_fr[8 * u + 2 * t]);
      fr[u][0] = both.x;
      fr[u][1] = both.y;
#pragma unroll
      for (int y = 0; y < 2; ++y) from[u][y] = -kNever, l[u][y] = 0.f;
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[u][j][k] = 0.f;
    }
#pragma unroll 1
    for (int k = 0; k < chunks; ++k) {
      asm volatile("cp.async.wait_group %0;" ::"n"(RING - 2) : "memory");
      __syncwarp();
      fetch();
      const uint32_t kt = get, vt = get + F::TILE;
      get = get + 2 * F::TILE == ring + RING * 2 * F::TILE ? ring : get + 2 * F::TILE;
      if (k >= valid) break;  // (the last one at most)
      // ---- scores
      float s[SUB][NT][4];  // slots 16 h + s0, 16 h + s1 of rows 2 t and 2 t + 1, in units of 1 / fr
#pragma unroll
      for (int h = 0; h < SUB; ++h) {
        uint32_t kw[2][NI], pr[2][4], own[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t rec = kt + (16 * h + (x ? s1 : s0)) * REC;
          if constexpr (NI == 4) {
            load4(kw[x], rec + t * 16);
          } else if constexpr (NI == 2) {
            load2(kw[x], rec + t * 8);
          } else {
#pragma unroll
            for (int b = 0; b < NI; ++b) kw[x][b] = load1(rec + (t * NI + b) * 4);
          }
          load4(pr[x], rec + 16 * NI);
          own[x] = load1(rec + 16 * NI + 4 * t);
        }
#pragma unroll
        for (int u = 0; u < NT; ++u) {
          const uint2 q = KEEP_Q ? qm[u] : sh_qm[u][lane];
          mma_new(s[h][u], own[0], own[1], own[0], own[1], q.x, q.y);
#pragma unroll
          for (int y = 0; y < 4; ++y) s[h][u][y] *= 0x1p-10f;
        }
#pragma unroll
        for (int grp = 0; grp < NG; ++grp) {
          const int b = NI > 2 ? grp : grp >> 1;
          float acc[NT][4];
#pragma unroll
          for (int e = NI > 2 ? 0 : grp & 1; e < (NI > 2 ? 2 : (grp & 1) + 1); ++e) {
            const uint32_t w0 = e ? kw[0][b] >> 8 : kw[0][b], w1 = e ? kw[1][b] >> 8 : kw[1][b];
#pragma unroll
            for (int y = 0; y < QP; ++y)
#pragma unroll
              for (int u = 0; u < NT; ++u) {
                const uint4 q = KEEP_Q ? qb[KEEP_Q ? u : 0][b] : sh_q[y][u][b][lane];
                const uint32_t b0 = e ? q.z : q.x, b1 = e ? q.w : q.y;
                if ((NI > 2 && e) || y)
                  mma_add(acc[u], w0 & 0x000f000fu, w1 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x00f000f0u, b0, b1);
                else
                  mma_new(acc[u], w0 & 0x000f000fu, w1 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x00f000f0u, b0, b1);
              }
          }
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float sc = __low2float(*reinterpret_cast<const __half2*>(&pr[x][grp]));
#pragma unroll
            for (int u = 0; u < NT; ++u)
#pragma unroll
              for (int y = 0; y < 2; ++y) s[h][u][2 * x + y] = fmaf(sc, acc[u][2 * x + y], s[h][u][2 * x + y]);
          }
        }
      }
      const bool whole = k >= k_lo && k < k_hi;
      if (!whole || a.scores) {
        const int tile = tile0 + k * NW;
        const bool in_a = tile < rt.ta;
        const int j0 = in_a ? rt.a0 + tile * TK : rt.b0 + (tile - rt.ta) * TK, jend = in_a ? rt.a1 : rt.b1;
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int m = 8 * u + 2 * t + y;
            const int pos = MULTI ? pos_first + (m0 + m) / group : pos_first;
            const int low = window_low(a, rt.start, pos);
#pragma unroll
            for (int x = 0; x < 2 * SUB; ++x) {
              const int h = x >> 1, j = j0 + 16 * h + (x & 1 ? s1 : s0);
              if (j >= jend || !slot_seen(a, rt.start, pos, low, j)) s[h][u][2 * (x & 1) + y] = -INFINITY;
              if (a.scores && j < jend && m < rows_here)
                a.scores[((int64_t)(p.r * a.kv_heads + head) * nG + m0 + m) * a.capacity + j] = s[h][u][2 * (x & 1) + y] * fr[u][y];
            }
          }
      }
      // ---- weights, by what exceeds the reference; past the slack it moves
      float z[SUB][NT][2][2], most = -INFINITY;
      auto shift = [&](const bool fused) {
#pragma unroll
        for (int h = 0; h < SUB; ++h)
#pragma unroll
          for (int u = 0; u < NT; ++u)
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
              for (int y = 0; y < 2; ++y)
                z[h][u][x][y] = fused ? fmaf(s[h][u][2 * x + y], fr[u][y], from[u][y])
                                      : __fadd_rn(__fmul_rn(s[h][u][2 * x + y], fr[u][y]), from[u][y]);
      };
      shift(true);
      if (huge) shift(false);
#pragma unroll
      for (int h = 0; h < SUB; ++h)
#pragma unroll
        for (int u = 0; u < NT; ++u) most = fmaxf(most, fmaxf(fmaxf(z[h][u][0][0], z[h][u][0][1]), fmaxf(z[h][u][1][0], z[h][u][1][1])));
      if (__any_sync(0xffffffffu, most > kMove)) {
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            float mx = -INFINITY;
#pragma unroll
            for (int h = 0; h < SUB; ++h) mx = fmaxf(mx, fmaxf(s[h][u][y], s[h][u][2 + y]));
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
            const float now = fminf(kRaise - __fmul_rn(mx, fr[u][y]), from[u][y]);
            const float by = now == from[u][y] ? 1.f : ex2(now - from[u][y]);
            from[u][y] = now;
            huge = huge || (fabsf(now) > 0x1p20f && now != -kNever);
            l[u][y] *= by;
#pragma unroll
            for (int j = 0; j < MT; ++j) {
              o[u][j][y] *= by;
              o[u][j][2 + y] *= by;
            }
          }
        huge = __any_sync(0xffffffffu, huge);
        shift(true);
        if (huge) shift(false);
      }
#pragma unroll
      for (int h = 0; h < SUB; ++h) {
        const uint32_t at_h = vt + 16 * h * REC;
        // As B operand of the values' product: slots of rows 0..7 and 8..15 of the tile's order (float16 outputs: and
        // what their rounding left).
        uint32_t pw[WP][NT][2];
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float w0 = ex2(z[h][u][x][0]), w1 = ex2(z[h][u][x][1]);
            l[u][0] += w0;
            l[u][1] += w1;
            if constexpr (FULL) {
              float2 rest = make_float2(w0, w1);
#pragma unroll
              for (int y = 0; y < 3; ++y) pw[y][u][x] = transposed(next_piece(rest));
              continue;
            }
            const uint32_t both = pack16(w0, w1);
            pw[0][u][x] = transposed(both);
            if constexpr (HALVES) {
              const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&both));
              pw[1][u][x] = transposed(pack16(w0 - h.x, w1 - h.y));
            }
          }
        // ---- values
        const uint32_t ra[4] = {at_h + va, at_h + vb, at_h + va + REC, at_h + vb + REC};
        uint32_t vw[4][NB], pr[4][2];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if constexpr (NI == 4) {
            load2(vw[x], ra[x] + g * 8);
            load2(pr[x], ra[x] + 16 * NI + (g & 1) * 8);
          } else if constexpr (NI == 3) {  // words 2 g, 2 g + 1 of twelve
            const int w = min(2 * g, 10);
            load2(vw[x], ra[x] + w * 4);
            pr[x][0] = load1(ra[x] + 16 * NI + w % 3 * 4);
            pr[x][1] = load1(ra[x] + 16 * NI + (w + 1) % 3 * 4);
          } else {
            const int w = NI == 2 ? g : g & 3;
            vw[x][0] = load1(ra[x] + w * 4);
            load2(pr[x], ra[x] + 16 * NI + w % NI * 8);
          }
        }
        uint32_t sc[2][2], mi[2][2];  // [rows 0..7, 8..15][group]
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            sc[x][y] = __byte_perm(pr[2 * x][y], pr[2 * x + 1][y], 0x5410);
            mi[x][y] = __byte_perm(pr[2 * x][y], pr[2 * x + 1][y], 0x7632);
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
            for (int y = 0; y < 2; ++y) {
              const uint32_t lo = (sc[x][y] & 0x7c00u) == 0x7c00u || (mi[x][y] & 0x7c00u) == 0x7c00u ? 0xffffu : 0u;
              const uint32_t hi = (sc[x][y] & 0x7c000000u) == 0x7c000000u || (mi[x][y] & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u;
              bad[x][y] = lo | hi;
              any |= bad[x][y];
              sc[x][y] &= ~bad[x][y];
              mi[x][y] &= ~bad[x][y];
            }
          hide = __any_sync(0xffffffffu, any != 0u);
        }
        // The value of nibble j (0..3) of a 16-bit half, of two slots side by side.
        auto value = [&](uint32_t w, int j, uint32_t scale, uint32_t mid) {
          const uint32_t x = j & 2 ? w >> 8 : w;
          const uint32_t c8 = j & 1 ? add16(and_or(x, k_odd, k_64), 0xd480d480u)      // 64 + c - 72
                                    : add16(and_or(x, k_even, k_1024), 0xe408e408u);  // 1024 + c - 1032
          return fma16(c8, scale, mid);
        };
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const uint32_t l0 = __byte_perm(vw[0][b], vw[1][b], 0x5410), h0 = __byte_perm(vw[0][b], vw[1][b], 0x7632);
          const uint32_t l1 = __byte_perm(vw[2][b], vw[3][b], 0x5410), h1 = __byte_perm(vw[2][b], vw[3][b], 0x7632);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int y = NI > 2 ? b : j >> 1;
            if constexpr (FULL) {
              uint32_t v[3][4];
              pieces(l0, j, sc[0][y], mi[0][y], v[0][0], v[1][0], v[2][0]);
              pieces(h0, j, sc[0][y], mi[0][y], v[0][1], v[1][1], v[2][1]);
              pieces(l1, j, sc[1][y], mi[1][y], v[0][2], v[1][2], v[2][2]);
              pieces(h1, j, sc[1][y], mi[1][y], v[0][3], v[1][3], v[2][3]);
              // The smallest products first; those below 2^-24 of the whole are left out.
#pragma unroll
              for (int z = 2; z >= 0; --z)
#pragma unroll
                for (int x = z; x >= 0; --x)
#pragma unroll
                  for (int u = 0; u < NT; ++u)
                    mma_bf16(o[u][4 * b + j], v[x][0], v[x][1], v[x][2], v[x][3], pw[z - x][u][0], pw[z - x][u][1]);
            } else {
              const uint32_t a0 = value(l0, j, sc[0][y], mi[0][y]), a1 = value(h0, j, sc[0][y], mi[0][y]);
              const uint32_t a2 = value(l1, j, sc[1][y], mi[1][y]), a3 = value(h1, j, sc[1][y], mi[1][y]);
#pragma unroll
              for (int z = 0; z < WP; ++z)
#pragma unroll
                for (int u = 0; u < NT; ++u) mma_add(o[u][4 * b + j], a0, a1, a2, a3, pw[z][u][0], pw[z][u][1]);
            }
          }
        }
        if (MULTI && hide) {
          // Ones where a row sees a slot, in the weights' place: weights may be zero.
          constexpr uint32_t one = FULL ? 0x3f803f80u : kOnes;
          const int tile = tile0 + k * NW;
          const bool in_a = tile < rt.ta;
          const int j0 = (in_a ? rt.a0 + tile * TK : rt.b0 + (tile - rt.ta) * TK) + 16 * h, jend = in_a ? rt.a1 : rt.b1;
          uint32_t sees[NT][2];
#pragma unroll
          for (int u = 0; u < NT; ++u)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int j = j0 + (x ? s1 : s0);
              uint32_t both = 0u;
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                const int pos = pos_first + (m0 + 8 * u + 2 * t + y) / group;
                if (j < jend && slot_seen(a, rt.start, pos, window_low(a, rt.start, pos), j)) both |= y ? one & 0xffff0000u : one & 0xffffu;
              }
              sees[u][x] = transposed(both);
            }
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int y = NI > 2 ? b : j >> 1;
              const uint32_t x0 = bad[0][y] & one, x1 = bad[1][y] & one;
#pragma unroll
              for (int u = 0; u < NT; ++u) {
                float seen[4];
                if constexpr (FULL) {
                  seen[0] = seen[1] = seen[2] = seen[3] = 0.f;
                  mma_bf16(seen, x0, x0, x1, x1, sees[u][0], sees[u][1]);
                } else {
                  mma_new(seen, x0, x0, x1, x1, sees[u][0], sees[u][1]);
                }
#pragma unroll
                for (int q = 0; q < 4; ++q)
                  if (seen[q] != 0.f) o[u][4 * b + j][q] = __int_as_float(0x7fc00000);
              }
            }
        }
      }
    }
    // The warp's results into shared memory.
#pragma unroll
    for (int u = 0; u < NT; ++u) {
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int m = 8 * u + 2 * t + y;
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[u][y] += __shfl_xor_sync(0xffffffffu, l[u][y], x);
        if (g == 0) {
          warp_m[warp][m] = -from[u][y];
          warp_l[warp][m] = l[u][y];
        }
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
    if (more) {
      const bool row_ends = p.h + 1 == K;
      load_q(row_ends ? p.r + 1 : p.r, row_ends ? 0 : p.h + 1);
    }
    __syncthreads();
    const bool alone = first >= c0 && end <= c1;
    const int slot = 2 * c + (first >= c0);
    if (tid < ROWS) {
      float top = -INFINITY, L = 0.f;
#pragma unroll
      for (int k = 0; k < NW; ++k) top = fmaxf(top, warp_m[k][tid]);
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        const float by = ex2(warp_m[k][tid] - top);
        factor[k][tid] = by;
        L = fmaf(warp_l[k][tid], by, L);
      }
      joined[tid] = make_float2(top, L);
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
    if (more) make_q();  // (nobody reads the queries past the barriers above)
    __syncthreads();
    last_shared = !alone;
    if (!more) break;
    // A unit that an earlier block began arrives at once: that block, which ends with it, mostly finds all there.
    if (!alone && tid == 0) sh_last[shared_parts - 1] = arrive_at(shared_part[shared_parts - 1]);
    p.k = 0;
    if (++p.h == K) {
      p.h = 0;
      before += p.chunks + between;
      p.row(a, p.r + 1);
    }
  }

  // ---- units shared with other blocks: who arrives last joins
  auto join = [&](const Shared& q, int c_first, int b0, int step, int count, bool last) {
    const int head = q.h / row_groups, m0 = (q.h - head * row_groups) * ROWS, rows_here = min(ROWS, nG - m0);
    auto slot_of = [&](int k) { return (int64_t)2 * (b0 + k * step) + (b0 + k * step == c_first); };
    // The first parts' values are on their way while their factors are made.
    constexpr int AHEAD = 16 / ITEMS > 6 ? 6 : 16 / ITEMS;
    float4 early[ITEMS][AHEAD];
    auto part_at = [&](int k, int x) {
      const int v = tid + x * THREADS, m = v / (OS / 4), d = (v - m * (OS / 4)) * 4;
      return __ldcg(reinterpret_cast<const float4*>(a.part_o + (slot_of(k) * ROWS + min(m, ROWS - 1)) * OS + d));
    };
#pragma unroll
    for (int x = 0; x < ITEMS; ++x)
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
        if (k < count) early[x][k] = part_at(k, x);
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
      auto add = [&](int k, float4 y) {
        const float by = factor[k][m];
        sum.x = fmaf(y.x, by, sum.x);
        sum.y = fmaf(y.y, by, sum.y);
        sum.z = fmaf(y.z, by, sum.z);
        sum.w = fmaf(y.w, by, sum.w);
      };
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
        if (k < count) add(k, early[x][k]);
#pragma unroll 4
      for (int k = AHEAD; k < count; ++k) add(k, part_at(k, x));
      if (last)
        write_out(q.r, head, m0 + m, d, sum, joined[m].y);
      else
        *reinterpret_cast<float4*>(a.part_o + (slot_of(0) * ROWS + m) * OS + d) = sum;
    }
  };
  if (tid == 0 && last_shared) sh_last[shared_parts - 1] = arrive_at(shared_part[shared_parts - 1]);
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

template <typename T, int NI, int NT, int SUB, int NW, int RING, bool MULTI>
cudaError_t record(const AttnArgs& a, int row_groups, cudaStream_t stream) {
  constexpr size_t smem = (size_t)NW * RING * 2 * Form<NI, SUB>::TILE + sizeof(float) * NW * 8 * NT * 32 * NI;
  const cudaError_t e = allow_smem<attn_record_kernel<T, NI, NT, SUB, NW, RING, MULTI>>(smem);
  if (e != cudaSuccess) return e;
  return launch_after(true, attn_record_kernel<T, NI, NT, SUB, NW, RING, MULTI>, dim3(kTokenBlocks), NW * 32, smem, stream, a,
                      kTokenBlocks, row_groups);
}

template <typename T, int NI, bool MULTI> cudaError_t record_rows(const AttnArgs& a, const RecordRows& x, cudaStream_t stream) {
  if constexpr (!std::is_same<T, float>::value) {
    // Tiles of 32 slots where blocks take many (679 cycles per 16 slots and scheduler, 798 with tiles of 16, when they came in); of
    // 16 where that gives each chunk of 128 slots a block, and a unit not more than 16 to be joined (two rows over 516 slots
    // 10.7 us, 12.0 with 32; one row over 4096 slots 17.7 us, 14.2 with 32).
    if (x.tiles == 2)
      return x.fits ? record<T, NI, 2, 1, 8, 5, MULTI>(a, x.groups, stream) : record<T, NI, 2, 2, 8, 3, MULTI>(a, x.groups, stream);
  }
  return record<T, NI, 1, 1, 12, 4, MULTI>(a, x.groups, stream);
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
  if (a.dtype == 0) return record_any<float>(a, x, stream);
  return a.dtype == 1 ? record_any<__half>(a, x, stream) : record_any<__nv_bfloat16>(a, x, stream);
}

}  // namespace sv
