// sv_attention_tile.cu -- attention of many query rows per key/value head (prompts,
// chunks of prompts, a batch over a shared prefix) on the fifth-generation tensor
// cores, float16 / bfloat16.
//
// A block (one per SM, taking pieces of work in turn) holds up to two tiles of 128 query rows (row m = query i * G + head g of one
// key/value head's group, so that a group's heads share every load) and walks 64-slot
// tiles of the keys and values.  Per row, in one pass: s_j = (q . k_j) scale log2 e,
// o += 2^(s_j - ref) v_j, l += 2^(s_j - ref).  ref is the running maximum, except that
// it moves only when a score exceeds it by more than 2^8 (the weights stay in range of
// float16), so that the output in tensor memory is rarely rescaled.
//
// Roles (12 warps):
//   warps 0-3, 4-7  one softmax group per query tile, one row per thread: scores from
//                   TMEM into registers, mask, exponentials, sums; the weights go back
//                   to TMEM in 16 bits over the scores they came from; at the end the
//                   division and the output
//   warp 8          TMA: keys and values in turn through a ring of eight 64-slot
//                   stages, 128-byte swizzle
//   warps 9, 10     the products of one query tile each, issued by one lane:
//                   S = Q K^T (both operands in shared memory) and O += P V (P in TMEM,
//                   V as it lies: MN-major).  Each tile has two score buffers: while its
//                   softmax works on one, its next scores form in the other.  One warp for
//                   both tiles took longer to issue than the products take
//   warp 11         values of tiles that not every row sees whole: zeros in slots past
//                   the end, and in place of what is not finite, which would reach
//                   rows that do not see it (0 * NaN); such slots are noted, and the
//                   rows that do see them get their values at the end
// TMEM: S0 (two buffers of 64 columns) | S1 | O0 | O1, 128 columns each; P overlays its
// S.  With one 128-slot score buffer per tile the chain softmax -> P V -> Q K^T -> softmax
// left the tensor cores idle half of the time (545 us for the 8192-token prompt).
//
// Every wait is bounded: a role that waits in vain sets the block's abort flag, all
// roles leave their loops, copies and products in flight are waited for (bounded), the
// TMEM is freed and the rows' outputs become NaN (status SV_ST_TIMEOUT).
#include <atomic>
#include <cstring>
#include <type_traits>

#include "../../include/starvector_sampling.h"
#include "sv_attention.h"
#include "sv_tcgen05.cuh"

namespace sv {
namespace {

constexpr int NT = 384;
constexpr int kSMs = 148;
constexpr int BM = 128, BN = 64;
constexpr int kMostRing = 4;       // steps (64 slots) whose keys and values are held
constexpr float kSlack = 8.f;
constexpr float kHuge = 0x1p20f;  // references whose last place is no longer small beside the slack

// kPlain: keys and values of the queries' type.  What a cache held in 4 bits stands for comes as float16:
// kHalves: for bfloat16 queries, which become float16 too, each row times a power of two (they lose nothing, and the
// keys an eighth of what bfloat16 would); kPairs: for float16 queries, each key and each weight as two float16, the
// second what the first one's rounding left (error of 4 x 100 queries against 64 bits: 0.00058 without, 0.00036 with the
// keys' alone; 0.00021 is the output's own rounding).
enum Source { kPlain, kHalves, kPairs };
constexpr int kEdges = 16;  // tiles that not every row of a block sees whole: at most twelve, see whole()

template <int DC, Source SRC> struct Layout {
  static constexpr int RING = SRC == kPairs && DC == 2 ? 3 : kMostRing, STAGES = 2 * RING;
  static constexpr uint32_t kQHalf = BM * 128, kHalf = BN * 128;  // 64 dimensions of a tile's rows
  static constexpr uint32_t kQTile = DC * kQHalf, kTile = DC * kHalf;
  static constexpr uint32_t kRing = 2 * kQTile;                      // after two query tiles
  static constexpr uint32_t kLow = kRing + STAGES * kTile;           // kPairs: the keys' second halves, one tile a step
  static constexpr uint32_t kBytes = kLow + (SRC == kPairs ? RING * kTile : 0) + 1024;  // alignment slack
};

struct Shared {
  // full, ready: a stage's copy, and its edge-tile pass.  s_full, pv_done: a query tile's scores of step j and
  // its product of step j (they also free the step's keys and values); one barrier for each of the steps
  // that the ring holds, so that none gets two phases ahead of who waits for it.
  uint64_t q_full[2], full[2 * kMostRing], ready[2 * kMostRing], s_full[2][kMostRing], p_full[2][2], pv_done[2][kMostRing],
      written[2], drained[2];
  float row_scale[2][BM];  // kHalves: of a row's scores
  float2 pair[BM];  // PAIRED: the second group's references and sums
  uint32_t tmem;
  uint32_t bad[kEdges][BN / 32];  // per edge tile: its slots with values that are not finite
  int bad_from[kEdges], any_bad;
  uint32_t limit_ns;  // of a wait
  volatile int abort;
};

struct Maps {
  CUtensorMap k, v, low;
  int32_t row_mul, head_mul;  // 0: all rows (heads) share one entry
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^x kept in its place among volatile instructions (within a group's turn).
__device__ __forceinline__ float ex2_here(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two f32 values as one operand of the packed FP32 instructions.
__device__ __forceinline__ uint64_t pack2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Named barriers 1 and 2: softmax group t waits for its turn, or passes it to the other.
__device__ __forceinline__ void turn_wait(int t) { asm volatile("bar.sync %0, 256;" ::"r"(1 + t) : "memory"); }
__device__ __forceinline__ void turn_pass(int t) { asm volatile("bar.arrive %0, 256;" ::"r"(2 - t) : "memory"); }

template <typename T> struct Half16;
template <> struct Half16<__half> {
  static constexpr bool bf16 = false;
  static constexpr uint32_t expo = 0x7c00u;
  __device__ static uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <> struct Half16<__nv_bfloat16> {
  static constexpr bool bf16 = true;
  static constexpr uint32_t expo = 0x7f80u;
  __device__ static uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

__device__ __forceinline__ void unpack8(const uint4& v, float (&x)[8]) {  // of bfloat16
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(h[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

// A bounded wait that also ends when another role has given up.
__device__ __noinline__ bool wait_slow(Shared& sh, uint32_t bar, uint32_t phase) {
  const uint64_t t0 = gtimer_ns();
  for (;;) {
    if (mbar_try(bar, phase)) return true;
    if (sh.abort) return false;
    if (gtimer_ns() - t0 > sh.limit_ns) {
      sh.abort = 1;
      return false;
    }
  }
}
__device__ __forceinline__ bool wait_one(Shared& sh, void* bar, uint32_t phase) {
  const uint32_t b = smem_u32(bar);
  return mbar_try(b, phase) || wait_slow(sh, b, phase);
}
// By a whole warp, with one verdict for all its lanes.
__device__ __forceinline__ bool wait(Shared& sh, void* bar, uint32_t phase) {
  return __all_sync(0xffffffffu, wait_one(sh, bar, phase));
}

// One piece of work: up to two query tiles of a unit over a share of its slots.
struct Item {
  int m0, mt, m_last;      // first query row, tiles that hold rows, last row
  int h, r, split;         // key/value head, cache row (own part), share of the slots
  int start, end;          // the row's slots
  int a0, a1, b0, b1, ta;  // [a0, a1) sinks before the window, [b0, b1) the rest; steps of the former
  int t0, nt;              // steps
};

// PAIRED: blocks of one query tile (and one item each), whose steps the two softmax groups
// and product warps take in turn, each with an output of its own, joined at the end.
// T: the queries' and the output's type; H: that of the products' operands.
template <typename T, int DC, bool PAIRED, Source SRC>
__global__ void __launch_bounds__(NT, 1) attn_tile_kernel(const __grid_constant__ AttnArgs a,
                                                          const __grid_constant__ Maps maps, const bool prefix,
                                                          const int tiles_m, const int units, const int items) {
  using L = Layout<DC, SRC>;
  using H = std::conditional_t<SRC == kPlain, T, __half>;
  constexpr int RING = L::RING, STAGES = L::STAGES;
  // Of a 4-bit cache: log2 of the weight that a new reference stands for, as in sv_attention_record.cu.
  constexpr float kRaise = SRC == kPlain ? 0.f : 7.f;
  static_assert(!PAIRED || RING % 2 == 0, "a group's every other step alternates a barrier's phase");
  constexpr int LPR = DC * 8, RPI = 32 / LPR;  // lanes of a row's 16-byte vectors, rows per warp instruction
  extern __shared__ unsigned char dyn_raw[];
  __shared__ Shared sh;
  unsigned char* dyn = dyn_raw + ((1024u - (smem_u32(dyn_raw) & 1023u)) & 1023u);
  launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nG = a.n * a.group;
  const int rows_m = prefix ? a.rows * nG : nG;
  const int S = prefix ? a.p_splits : max(a.o_splits, 1);
  const int blocks_m = items / (S * units);

  // The last rows see the most slots under a causal mask: they come first.
  auto item_at = [&](int w) {
    Item it;
    const int unit = w % units, x = w / units;
    it.split = x % S;
    it.m0 = (blocks_m - 1 - x / S) * tiles_m * BM;
    it.mt = min(tiles_m, (rows_m - it.m0 + BM - 1) / BM);
    it.m_last = min(it.m0 + tiles_m * BM, rows_m) - 1;
    it.h = prefix ? unit : unit % a.kv_heads;
    it.r = prefix ? 0 : unit / a.kv_heads;
    it.start = it.a0 = it.a1 = it.b0 = 0;
    it.end = it.b1 = a.prefix;
    if (!prefix) {
      const RowSpan sp = row_span(a, it.r);
      it.start = sp.start;
      it.end = sp.end;
      const int pf = sp.end - a.n + it.m0 / a.group, pl = sp.end - a.n + it.m_last / a.group;
      it.b0 = window_low(a, sp.start, pf);
      it.b1 = pl < sp.start ? it.b0 : max(pl + 1, it.b0);
      it.a0 = sp.start;
      it.a1 = pl >= sp.start ? max(it.a0, min(sp.start + a.sinks, it.b0)) : it.a0;
    }
    it.ta = (it.a1 - it.a0 + BN - 1) / BN;
    const int steps = it.ta + (it.b1 - it.b0 + BN - 1) / BN;
    it.t0 = (int)((int64_t)steps * it.split / S);
    it.nt = (int)((int64_t)steps * (it.split + 1) / S) - it.t0;
    return it;
  };
  auto tile_at = [](const Item& it, int j, int& j0, int& jend) {
    const int t = it.t0 + j;
    j0 = t < it.ta ? it.a0 + t * BN : it.b0 + (t - it.ta) * BN;
    jend = t < it.ta ? it.a1 : it.b1;
  };
  // How many 16-slot products a step's values need: the rest of its tile is not read.
  auto value_blocks = [](int j0, int jend) { return min(BN / 16, (jend - j0 + 15) / 16); };
  // The steps whose slots rows [first, last] all see: j < a_whole (sinks) or w0 <= j < w1.
  struct Whole {
    int a_whole, w0, w1;
    int from, to;  // the window's slots that all of them see
    __device__ __forceinline__ bool operator()(int j) const { return j < a_whole || (j >= w0 && j < w1); }
  };
  auto whole_steps = [&](const Item& it, int first, int last) {
    const int from = prefix ? it.b0 : window_low(a, it.start, it.end - a.n + last / a.group);
    const int to = prefix ? it.b1 : min(it.b1, it.end - a.n + first / a.group + 1);
    const int b = it.ta - it.t0;  // the window's first step
    Whole x;
    x.from = from;
    x.to = to;
    x.a_whole = (it.a1 - it.a0) / BN - it.t0;
    x.w0 = b + (max(from - it.b0, 0) + BN - 1) / BN;
    x.w1 = b + max(to - it.b0, 0) / BN;
    return x;
  };

  // A softmax warp reads and writes its 32 rows of queries and output RPI rows at a time,
  // LPR lanes to a row: row my_row + k RPI for this lane, its vector my_vec.
  const int my_row = (warp & 3) * 32 + lane / LPR, my_vec = lane % LPR;
  const int wg = warp >> 2;                   // a softmax warp's query tile
  unsigned char* qb = dyn + wg * L::kQTile;  // its queries, and at the end its output on the way out
  auto q_vec = [&](int row, int vec) {
    return reinterpret_cast<uint4*>(qb + (vec >> 3) * L::kQHalf + row * 128 + (((vec & 7) ^ (row & 7)) << 4));
  };
  const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;  // a negative scale turns the queries' signs
  auto load_queries = [&](const Item& it) {
    uint4 v[LPR];
    int m = it.m0 + wg * BM + my_row;
    int r = prefix ? m / nG : it.r, i = prefix ? m - r * nG : m, g = i;
    i /= a.group;
    g -= i * a.group;
    const T* src = static_cast<const T*>(a.q) + r * a.q_row + i * a.q_tok + (int64_t)(it.h * a.group + g) * a.q_head +
                   my_vec * 8;
    const int64_t step = RPI * a.q_head, next_query = a.q_tok - a.group * a.q_head, next_row = a.q_row - a.n * a.q_tok;
#pragma unroll
    for (int k = 0; k < LPR; ++k, m += RPI) {
      v[k] = m < rows_m && my_vec * 8 < a.dim ? __ldg(reinterpret_cast<const uint4*>(src)) : make_uint4(0u, 0u, 0u, 0u);
      src += step;
      for (g += RPI; g >= a.group; g -= a.group) {
        src += next_query;
        if (++i == a.n) i = 0, src += next_row;  // (without a prefix: past the last row, not read)
      }
    }
#pragma unroll
    for (int k = 0; k < LPR; ++k) {
      if constexpr (SRC == kHalves) {
        float x[8], most = 0.f;
        unpack8(v[k], x);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (fabsf(x[e]) < INFINITY) most = fmaxf(most, fabsf(x[e]));
#pragma unroll
        for (int e = 1; e < LPR; e <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, e));
        // The row's largest value to [2^14, 2^15), with the scale's sign.
        const int ex = max(15, (int)(__float_as_uint(most) >> 23));
        const float up = copysignf(__uint_as_float((uint32_t)(268 - min(ex, 254)) << 23), a.scale);
        v[k] = make_uint4(Half16<H>::pack(x[0] * up, x[1] * up), Half16<H>::pack(x[2] * up, x[3] * up),
                          Half16<H>::pack(x[4] * up, x[5] * up), Half16<H>::pack(x[6] * up, x[7] * up));
        // (Zero would make NaN of hidden slots' -infinity; past 2^89 scores could leave f32, and any two that differ are
        // 2^41 apart by then.)
        if (my_vec == 0)
          sh.row_scale[wg][my_row + k * RPI] =
              fminf(fmaxf(fabsf(a.scale) * __uint_as_float((uint32_t)(min(ex, 254) - 14) << 23), 0x1p-126f), 0x1p89f);
      } else {
        v[k].x ^= flip, v[k].y ^= flip, v[k].z ^= flip, v[k].w ^= flip;
      }
      *q_vec(my_row + k * RPI, my_vec) = v[k];
    }
    if (SRC == kHalves) __syncwarp();
    fence_proxy_async_smem();
  };

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.q_full[i], 128);
      mbar_init(&sh.written[i], 128);
      mbar_init(&sh.drained[i], 1);
      for (int k = 0; k < 2; ++k) mbar_init(&sh.p_full[i][k], 128);
      for (int k = 0; k < RING; ++k) {
        mbar_init(&sh.s_full[i][k], 1);
        mbar_init(&sh.pv_done[i][k], 1);
      }
    }
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.ready[i], 1);
    }
    sh.any_bad = 0;
    sh.limit_ns = a.test_head ? 2000000u : 2000000000u;
    for (int i = 0; i < kEdges; ++i)
      for (int k = 0; k < BN / 32; ++k) sh.bad[i][k] = 0;
    sh.abort = 0;
    mbar_init_fence();
  }
  if (warp == 9) tmem_alloc512(&sh.tmem);
  Item it = item_at(blockIdx.x);  // the grid has at most one block per item
  if (wg < it.mt && it.nt > 0) load_queries(it);
  tcgen05_before_sync();
  __syncthreads();
  tcgen05_after_sync();
  const uint32_t tmem = sh.tmem;

  // Steps are numbered through all the block's items: J = base + j.  Step J's keys and
  // values are in stages 2 J and 2 J + 1 (mod STAGES).  A query tile's scores alternate
  // between its two buffers (PAIRED: by its own count P of steps, every other one).
  if (warp == 8) {
    // ------------------------------------------------------------- copies
    if (lane == 0) {
      tma_prefetch_map(&maps.k);
      tma_prefetch_map(&maps.v);
      if (SRC == kPairs) tma_prefetch_map(&maps.low);
      int issued = 0;
      bool ok = true;
      for (int w = blockIdx.x; ok && w < items; w += gridDim.x) {
        if (w != (int)blockIdx.x) it = item_at(w);
        for (int x = 0; x < 2 * it.nt; ++x, ++issued) {
          const int st = issued % STAGES, step = (issued >> 1) % RING;
          // Free once all tiles' products of four steps ago are done.
          for (int t = PAIRED ? (x >> 1) & 1 : 0; t < (PAIRED ? ((x >> 1) & 1) + 1 : tiles_m) && issued >= STAGES; ++t)
            ok = ok && wait_one(sh, x & 1 ? &sh.pv_done[t][step] : &sh.s_full[t][step], (issued / STAGES - 1) & 1);
          if (!ok) break;
          int j0, jend;
          tile_at(it, x >> 1, j0, jend);
          const bool low = SRC == kPairs && !(x & 1);
          mbar_expect_tx(&sh.full[st], low ? 2 * L::kTile : L::kTile);
          const CUtensorMap* map = x & 1 ? &maps.v : &maps.k;
#pragma unroll
          for (int d = 0; d < DC; ++d)
            tma_load4(dyn + L::kRing + st * L::kTile + d * L::kHalf, map, d * 64, j0, it.h * maps.head_mul,
                      it.r * maps.row_mul, &sh.full[st]);
          if (low)
#pragma unroll
            for (int d = 0; d < DC; ++d)
              tma_load4(dyn + L::kLow + step * L::kTile + d * L::kHalf, &maps.low, d * 64, j0, it.h * maps.head_mul,
                        it.r * maps.row_mul, &sh.full[st]);
        }
      }
      // Nothing may still be landing when the block ends.  (Without an abort its steps wait for it
      // anyway; one may still come after this point.)
      for (int i = max(0, issued - STAGES); i < issued; ++i) mbar_wait(&sh.full[i % STAGES], (i / STAGES) & 1);
    }
  } else if (warp == 9 || warp == 10) {
    // ------------------------------------------------------------- products
    constexpr uint32_t wqk = mma_word(Half16<H>::bf16, BN, false), wpv = mma_word(Half16<H>::bf16, 64 * DC, true);
    constexpr uint32_t kStep = L::kTile >> 4, kQStep = L::kQTile >> 4;
    const int t = warp - 9;
    const bool leader = elect_one();
    // Descriptors are sums of a base and constants, and what the loops depend on comes from
    // reductions, whose results the compiler knows to be the same in all lanes: otherwise
    // every product would first move its operands to uniform registers.
    const uint32_t tm = __reduce_max_sync(0xffffffffu, tmem);
    const uint32_t s_at = tm + t * 128, o_at = tm + 256 + t * 128;
    const uint64_t qd = smem_desc(smem_u32(dyn), 16) + (PAIRED ? 0 : t * kQStep);
    const uint64_t k_desc = smem_desc(smem_u32(dyn) + L::kRing, 16),
                   v_desc = smem_desc(smem_u32(dyn) + L::kRing, L::kHalf),
                   low_desc = smem_desc(smem_u32(dyn) + L::kLow, 16);
    // One lane waits and issues.  After an abort its waits fail at once and the rest of the
    // loop computes on what is there, which nobody uses.
    auto qk = [&](int J, int P) {
      const uint64_t kd = k_desc + (2 * J) % STAGES * kStep;
#pragma unroll
      for (int k = 0; k < 4 * DC; ++k)
        mma_ss(s_at + (P & 1) * BN, qd + (((k >> 2) * L::kQHalf + (k & 3) * 32) >> 4),
               kd + (((k >> 2) * L::kHalf + (k & 3) * 32) >> 4), wqk, k != 0);
      if constexpr (SRC == kPairs) {
        const uint64_t ld = low_desc + J % RING * kStep;
#pragma unroll
        for (int k = 0; k < 4 * DC; ++k)
          mma_ss(s_at + (P & 1) * BN, qd + (((k >> 2) * L::kQHalf + (k & 3) * 32) >> 4),
                 ld + (((k >> 2) * L::kHalf + (k & 3) * 32) >> 4), wqk, true);
      }
      mma_commit(&sh.s_full[t][J % RING]);
    };
    int base_ = 0, queries = 0;
    if (PAIRED) {
      const int steps = __reduce_max_sync(0xffffffffu, it.nt);
      if (leader && t < steps) {
        wait_one(sh, &sh.q_full[0], 0);
        for (int j = t; j < min(steps, t + 4); j += 2) {
          wait_one(sh, &sh.full[2 * j], 0);
          qk(j, j >> 1);
        }
      }
      __syncwarp();
#pragma unroll 1
      for (int c = 0; 2 * c + t < steps; ++c) {
        const int j = 2 * c + t, vi = 2 * j + 1, ki = 2 * j + 8;
        int j0, jend;
        tile_at(it, j, j0, jend);
        const int blocks = value_blocks(j0, jend);
        if (leader) {
          wait_one(sh, &sh.ready[vi % STAGES], (vi / STAGES) & 1);
          wait_one(sh, &sh.p_full[t][c & 1], (c >> 1) & 1);
          tcgen05_after_sync();
          const uint64_t vd = v_desc + (vi % STAGES) * kStep;
#pragma unroll
          for (int k = 0; k < BN / 16; ++k)
            if (k < blocks) mma_ts(o_at, s_at + (c & 1) * BN + k * 8, vd + k * (2048 >> 4), wpv, c != 0 || k != 0);
          if (SRC == kPairs)
#pragma unroll
            for (int k = 0; k < BN / 16; ++k)
              if (k < blocks) mma_ts(o_at, s_at + (c & 1) * BN + 32 + k * 8, vd + k * (2048 >> 4), wpv, true);
          mma_commit(&sh.pv_done[t][j % RING]);
          if (j + 4 < steps) {
            wait_one(sh, &sh.full[ki % STAGES], (ki / STAGES) & 1);
            qk(j + 4, c + 2);
          }
        }
        __syncwarp();
      }
    }
    for (int w = blockIdx.x; !PAIRED && w < items && t < tiles_m; w += gridDim.x) {
      if (w != (int)blockIdx.x) it = item_at(w);
      const int steps = __reduce_max_sync(0xffffffffu, it.nt);
      const int base = __reduce_max_sync(0xffffffffu, base_);
      if (t >= it.mt) {  // no rows: the stages are passed on as they come, through the softmax group
        if (leader)
          for (int J = base; J < base + steps; ++J) {
            wait_one(sh, &sh.full[(2 * J) % STAGES], (2 * J / STAGES) & 1);
            mma_commit(&sh.s_full[t][J % RING]);
            wait_one(sh, &sh.ready[(2 * J + 1) % STAGES], ((2 * J + 1) / STAGES) & 1);
            wait_one(sh, &sh.p_full[t][J & 1], (J >> 1) & 1);
            mma_commit(&sh.pv_done[t][J % RING]);
          }
        __syncwarp();
        base_ += steps;
        continue;
      }
      if (leader && steps > 0) {
        wait_one(sh, &sh.q_full[t], queries & 1);
        for (int j = 0; j < min(steps, 2); ++j) {
          wait_one(sh, &sh.full[(2 * (base + j)) % STAGES], (2 * (base + j) / STAGES) & 1);
          qk(base + j, base + j);
        }
      }
      queries += steps > 0;
      __syncwarp();
#pragma unroll 1
      for (int j = 0; j < steps; ++j) {
        const int J = base + j, vi = 2 * J + 1, ki = 2 * J + 4;
        int j0, jend;
        tile_at(it, j, j0, jend);
        const int blocks = value_blocks(j0, jend);
        if (leader) {
          wait_one(sh, &sh.ready[vi % STAGES], (vi / STAGES) & 1);
          wait_one(sh, &sh.p_full[t][J & 1], (J >> 1) & 1);
          tcgen05_after_sync();
          const uint64_t vd = v_desc + (vi % STAGES) * kStep;
#pragma unroll
          for (int k = 0; k < BN / 16; ++k)
            if (k < blocks) mma_ts(o_at, s_at + (J & 1) * BN + k * 8, vd + k * (2048 >> 4), wpv, j != 0 || k != 0);
          if (SRC == kPairs)
#pragma unroll
            for (int k = 0; k < BN / 16; ++k)
              if (k < blocks) mma_ts(o_at, s_at + (J & 1) * BN + 32 + k * 8, vd + k * (2048 >> 4), wpv, true);
          mma_commit(&sh.pv_done[t][J % RING]);
          if (j + 2 < steps) {
            wait_one(sh, &sh.full[ki % STAGES], (ki / STAGES) & 1);
            qk(J + 2, J + 2);
          }
        }
        __syncwarp();
      }
      base_ += steps;
      if (__any_sync(0xffffffffu, sh.abort)) break;
    }
    if (__any_sync(0xffffffffu, sh.abort)) {  // the products in flight
      if (leader) {
        mma_commit(&sh.drained[t]);
        mbar_wait(&sh.drained[t], 0);
      }
      __syncwarp();
    }
  } else if (warp == 11) {
    // ------------------------------------------------------------- values of edge tiles
    // Before an item's notes are made those of the item before have to be read: by the groups
    // that had rows and steps in it, no others.  Such a group cannot end its next item before
    // this warp has let that item's steps go, so it is never two phases ahead of a wait here.
    int base = 0, read_by = 0, phases[2] = {0, 0};  // the groups that read the item before's notes
    bool ok = true;
    for (int w = blockIdx.x; ok && w < items; w += gridDim.x) {
      if (w != (int)blockIdx.x) it = item_at(w);
      if (it.nt <= 0) continue;  // no steps, no notes
      if (read_by > 0) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (t < read_by) ok = ok && wait(sh, &sh.written[t], phases[t]++ & 1);
        if (!ok) break;
        if (sh.any_bad) {
          __syncwarp();
          for (int i = lane; i < kEdges * (BN / 32); i += 32) sh.bad[i / (BN / 32)][i % (BN / 32)] = 0;
          sh.any_bad = 0;
          __syncwarp();
        }
      }
      read_by = it.mt;
      int edge = 0;
      const Whole whole = whole_steps(it, it.m0, it.m_last);
      for (int j = 0; j < it.nt; ++j) {
        const int vi = 2 * (base + j) + 1, st = vi % STAGES;
        ok = wait(sh, &sh.full[st], (vi / STAGES) & 1);
        if (!ok) break;
        if (!whole(j)) {
          int j0, jend;
          tile_at(it, j, j0, jend);
          unsigned char* vb = dyn + L::kRing + st * L::kTile;
          // Only slots that some row does not see are looked at (sinks before the window are seen
          // by all), and behind the last slot those of its product are zeroed: where a block has
          // few queries that is a small part of the tile, and the steps wait for this warp
          // (looking at the whole tile, 4 x 100 queries of 64 dimensions took 31.9 us, now
          // 26.8; 3 x 577 of 128 20.2 and 16.9, the 8192-token prompt 443 and 413).  The swizzle permutes 16-byte vectors within
          // a slot only.
          const bool sink = it.t0 + j < it.ta;
          const int n = min(jend - j0, BN), last = 16 * value_blocks(j0, jend);
          const int seen0 = sink ? 0 : min(max(whole.from - j0, 0), n), seen1 = sink ? n : min(max(whole.to - j0, seen0), n);
          auto look = [&](int r0, int r1) {
            constexpr uint32_t E = Half16<H>::expo * 0x10001u;
            constexpr int kAhead = 4;  // vectors of a lane in flight
#pragma unroll 1
            for (int d = 0; d < DC; ++d) {
              uint4* vd = reinterpret_cast<uint4*>(vb + d * L::kHalf);
#pragma unroll 1
              for (int x0 = r0 * 8 + lane; x0 < r1 * 8; x0 += 32 * kAhead) {
                uint4 v[kAhead];
                uint32_t any = 0;
#pragma unroll
                for (int k = 0; k < kAhead; ++k) v[k] = vd[min(x0 + 32 * k, r1 * 8 - 1)];
                // A half with all exponent bits set leaves zero, and the subtraction its sign.
#pragma unroll
                for (int k = 0; k < kAhead; ++k)
                  any |= (((v[k].x & E) ^ E) - 0x10001u) | (((v[k].y & E) ^ E) - 0x10001u) |
                         (((v[k].z & E) ^ E) - 0x10001u) | (((v[k].w & E) ^ E) - 0x10001u);
                if (!(any & 0x80008000u)) continue;
                for (int k = 0; k < kAhead && x0 + 32 * k < r1 * 8; ++k) {
                  const int x = x0 + 32 * k;
                  uint32_t* w = reinterpret_cast<uint32_t*>(vd + x);
                  bool bad = false;
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    const uint32_t e = w[i] & E, lo = (e & 0xffffu) == (E & 0xffffu) ? 0xffffu : 0u,
                                   hi = (e & 0xffff0000u) == (E & 0xffff0000u) ? 0xffff0000u : 0u;
                    if (lo | hi) w[i] &= ~(lo | hi), bad = true;
                  }
                  if (bad) {
                    atomicOr(&sh.bad[edge][x >> 8], 1u << ((x >> 3) & 31));
                    sh.bad_from[edge] = j0;
                    sh.any_bad = 1;
                  }
                }
              }
            }
          };
          look(0, seen0);
          look(seen1, n);
          for (int x = n * 8 + lane; x < last * 8; x += 32)
#pragma unroll
            for (int d = 0; d < DC; ++d)
              *reinterpret_cast<uint4*>(vb + d * L::kHalf + x * 16) = make_uint4(0u, 0u, 0u, 0u);
          __syncwarp();
          fence_proxy_async_smem();
          edge = min(edge + 1, kEdges - 1);
        }
        __syncwarp();
        if (lane == 0 && it.h + 1 != a.test_head) mbar_arrive(&sh.ready[st]);
      }
      base += it.nt;
    }
  } else {
    // ------------------------------------------------------------- softmax and output
    const int t = wg, row = tid & 127;
    const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);
    const uint32_t o_at = lanes + 256 + t * 128;
    const bool direct = !prefix && a.o_splits == 0;
    const int64_t all = (int64_t)a.rows * a.kv_heads * nG;
    // After an abort the groups go through their steps all the same (on scores that nobody
    // uses), so that neither waits for a turn that does not come.
    if (t == 1 && (PAIRED || tiles_m == 2)) turn_pass(1);
    int base = 0;
    for (int w = blockIdx.x; w < items; w += gridDim.x) {
      if (w != (int)blockIdx.x) {
        it = item_at(w);
        if (t < it.mt && it.nt > 0) load_queries(it);
      }
      float ref = -INFINITY, l = 0.f;
      bool ok = true;
      // (With two groups at one query tile there is one item, whose rows' scales all threads saw at the start.)
      const float scale = SRC == kHalves ? sh.row_scale[PAIRED ? 0 : t][row] : fabsf(a.scale);
      const int mfirst = it.m0 + (PAIRED ? 0 : t * BM), mlast = min(mfirst + BM, rows_m) - 1, m = mfirst + row;
      const int pos = prefix ? a.prefix : it.end - a.n + m / a.group, low = prefix ? 0 : window_low(a, it.start, pos);
      // The item's rows are neighbours in the partial results (per head, for the prefix: all
      // cache rows' queries).
      const int64_t part_row = it.split * all + (int64_t)(prefix ? it.h : it.r * a.kv_heads + it.h) * rows_m;
      const bool both = PAIRED || it.mt == 2;
      if ((PAIRED || t < it.mt) && it.nt > 0) {
        if (t < it.mt) mbar_arrive(&sh.q_full[t]);
        const Whole whole = whole_steps(it, mfirst, mlast);
        const int rounds = PAIRED ? (it.nt + 1) >> 1 : it.nt;
        for (int own = 0; own < rounds; ++own) {
          const int j = PAIRED ? 2 * own + t : own, J = base + j, P = PAIRED ? own : J;
          if (PAIRED && j >= it.nt) {  // an odd step out: the other group's
            turn_wait(t);
            turn_pass(t);
            continue;
          }
          ok = ok && wait(sh, &sh.s_full[t][J % RING], (J / RING) & 1);
          tcgen05_after_sync();
          const uint32_t s_at = lanes + t * 128 + (P & 1) * BN;
          float s[BN];
          tmem_load64(s_at, s);
          const bool all_seen = whole(j);
          if (!all_seen) {
            int j0, jend;
            tile_at(it, j, j0, jend);
            const int r1 = min(pos + 1, jend) - j0, r0 = low - j0,
                      s1 = min(it.start + a.sinks, min(pos + 1, jend)) - j0;
#pragma unroll
            for (int c = 0; c < BN; ++c)
              if (!(c < r1 && (c >= r0 || c < s1))) s[c] = -INFINITY;
          }
          float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
          for (int c = 4; c < BN; c += 8) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mx[k] = max_nan(max_nan(mx[k], s[c + k]), c + 4 + k < BN ? s[(c + 4 + k) % BN] : mx[k]);
          }
          // A NaN stays in the maximum, so that it makes the whole row NaN.
          const float top = max_nan(max_nan(mx[0], mx[1]), max_nan(mx[2], mx[3])) * scale;
          const bool need = !(fabsf(ref) > kHuge ? top - ref <= kSlack + kRaise : top <= ref + (kSlack + kRaise)) && top != -INFINITY;
          if (__any_sync(0xffffffffu, need)) {
            const float f = need ? ex2(ref - (top - kRaise)) : 1.f;
            if (need) ref = top - kRaise;
            l *= f;
            if (own > 0) {  // the product before must be in, and this step's waits for these weights
              constexpr int back = PAIRED ? 2 : 1;
              ok = ok && wait(sh, &sh.pv_done[t][(J - back) % RING], ((J - back) / RING) & 1);
              tcgen05_after_sync();
#pragma unroll 1
              for (int d = 0; d < 64 * DC; d += 32) {
                float o[32];
                tmem_load32(o_at + d, o);
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] *= f;
                tmem_store32(o_at + d, o);
              }
            }
          }
          // Nothing seen yet: weights of zero; a maximum of +inf: NaN, as inf - inf.
          const float at = ref == -INFINITY ? 0.f : (ref == INFINITY ? __int_as_float(0x7fc00000) : ref);
          // Scores past kHuge are rounded as their maximum was: the fused product would set that maximum itself far off.
          float by = scale;
          if (fabsf(ref) > kHuge) {
#pragma unroll
            for (int c = 0; c < BN; ++c) s[c] *= scale;
            by = 1.f;
          }
          const uint64_t scale2 = pack2(by, by), at2 = pack2(-at, -at);
          uint64_t sum[2] = {0, 0}, z[BN / 2];
#pragma unroll
          for (int k = 0; k < BN / 2; ++k) z[k] = fma2(pack2(s[2 * k], s[2 * k + 1]), scale2, at2);
          // The special function unit takes 8 cycles for a warp's 32 exponentials, which is what
          // bounds a step: the two groups take turns at it, so that one is always busy with
          // its other work (when they came in, 445 us for the 8192-token prompt with and 470 us without them).  Moving
          // exponentials to the FP32 pipes by a polynomial (one pair in eight, or in four) took
          // 2 to 4 % longer: those pipes do the scaling and the sums already.
          uint32_t p[32];
          if (both) turn_wait(t);
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            float x, y;
            unpack2(z[k], x, y);
            x = ex2_here(x);
            y = ex2_here(y);
            sum[k & 1] = add2(sum[k & 1], pack2(x, y));
            p[k] = Half16<H>::pack(x, y);
            if constexpr (SRC == kPairs) {  // over the scores' place: what the rounding left, behind the weights
              const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&p[k]));
              s[k] = __uint_as_float(Half16<H>::pack(x - h.x, y - h.y));
            }
          }
          tmem_store32(s_at, p);
          if constexpr (SRC == kPairs) {
#pragma unroll
            for (int k = 0; k < 32; ++k) p[k] = __float_as_uint(s[k]);
            tmem_store32(s_at + 32, p);
          }
          if (both) turn_pass(t);
          float sx, sy;
          unpack2(add2(sum[0], sum[1]), sx, sy);
          l += sx + sy;
          tmem_wait_store();
          tcgen05_before_sync();
          mbar_arrive(&sh.p_full[t][P & 1]);
        }
      } else if (!PAIRED && t < tiles_m) {
        // No rows: step by step all the same.  A group that went ahead to its next item could
        // take an older phase of that item's barriers for the one it waits for.
        for (int j = 0; j < it.nt; ++j) {
          const int J = base + j;
          wait(sh, &sh.s_full[t][J % RING], (J / RING) & 1);
          mbar_arrive(&sh.p_full[t][J & 1]);
        }
      }
      base += it.nt;
      const int last = PAIRED ? ((it.nt - 1 - t) & ~1) + t : base - 1;  // this group's last step
      float f0 = 1.f, f1 = 0.f;                                         // PAIRED: the two outputs' factors
      bool second = false;
      if ((PAIRED ? last >= 0 && it.nt > t : t < it.mt && it.nt > 0) && ok) {
        ok = wait(sh, &sh.pv_done[t][last % RING], (last / RING) & 1);
        tcgen05_after_sync();
      }
      if (PAIRED) {
        if (t == 1) sh.pair[row] = make_float2(ref, ok ? l : __int_as_float(0x7fc00000));
        tcgen05_before_sync();
        asm volatile("bar.sync 3, 256;" ::: "memory");
        tcgen05_after_sync();
        if (t == 0) {
          const float2 other = sh.pair[row];
          const float top = fmaxf(ref, other.x), at = top == -INFINITY ? 0.f : top;
          second = it.nt > 1;
          f0 = ex2(ref - at);
          f1 = ex2(other.x - at);
          l = second ? l * f0 + other.y * f1 : l * f0;
          ref = top;
        }
      }
      if (t < it.mt) {
        ok = __all_sync(0xffffffffu, ok && !sh.abort);
        // (Rows of an item without steps may meet another item's notes, and see none of their slots.)
        const bool any_bad = *static_cast<volatile int*>(&sh.any_bad) != 0;
        const float inv = !ok ? __int_as_float(0x7fc00000) : (l == 0.f ? 0.f : (direct ? 1.f / l : 1.f));
#pragma unroll 1
        for (int c = 0; c < 64 * DC; c += 32) {
          float o[32];
          if (ok && it.nt > 0) {
            tmem_load32(o_at + c, o);
            if (PAIRED) {
              if (second) {
                float o1[32];
                tmem_load32(o_at + 128 + c, o1);
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = o[k] * f0 + o1[k] * f1;
              } else {
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] *= f0;
              }
            }
          } else {
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = 0.f;
          }
          if (any_bad && m < rows_m) {  // values that are not finite, for the rows that see them
            for (int e = 0; e < kEdges * BN; ++e) {
              if (!(sh.bad[e / BN][(e % BN) >> 5] >> (e & 31) & 1u)) continue;
              const int slot = sh.bad_from[e / BN] + e % BN;
              if (!prefix && !slot_seen(a, it.start, pos, low, slot)) continue;
              const H* vp = static_cast<const H*>(prefix ? a.pv : a.v) +
                            (prefix ? it.h * a.p_head + slot * a.p_slot
                                    : it.r * a.kv_row + it.h * a.kv_head + slot * a.kv_slot);
#pragma unroll
              for (int k = 0; k < 32; k += 8) {
                float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                if (c + k < a.dim) load8(vp + c + k, v);
#pragma unroll
                for (int x = 0; x < 8; ++x)
                  if (!isfinite(v[x])) o[k + x] += v[x];
              }
            }
          }
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] *= inv;
          // Through the queries' place (the products that read it are done): a thread writes
          // its row, then the lanes of a row write it out together.  16-bit rows go out whole,
          // f32 ones 32 DC dimensions at a time.
          bool flush;
          if (direct) {
#pragma unroll
            for (int k = 0; k < 32; k += 8)
              *q_vec(row, (c + k) >> 3) = make_uint4(Half16<T>::pack(o[k], o[k + 1]), Half16<T>::pack(o[k + 2], o[k + 3]),
                                                     Half16<T>::pack(o[k + 4], o[k + 5]), Half16<T>::pack(o[k + 6], o[k + 7]));
            flush = c + 32 == 64 * DC;
          } else {
#pragma unroll
            for (int k = 0; k < 32; k += 4)
              *q_vec(row, ((c % (32 * DC)) + k) >> 2) =
                  make_uint4(__float_as_uint(o[k]), __float_as_uint(o[k + 1]), __float_as_uint(o[k + 2]),
                             __float_as_uint(o[k + 3]));
            flush = (c + 32) % (32 * DC) == 0;
          }
          __syncwarp();
          if (flush) {
            const int d = direct ? my_vec * 8 : c + 32 - 32 * DC + my_vec * 4;
            int mm = mfirst + my_row, g = mm % a.group;
            T* out = static_cast<T*>(a.out) +
                     (((int64_t)it.r * a.n + mm / a.group) * a.heads + it.h * a.group + g) * a.dim + d;
            float* part = (prefix ? a.prefix_o : a.part_o) + (part_row + mm) * a.dim + d;
            const int64_t next_query = (int64_t)(a.heads - a.group) * a.dim;
#pragma unroll 4
            for (int k = 0; k < LPR; ++k, mm += RPI) {
              const uint4 v = *q_vec(my_row + k * RPI, my_vec);
              const bool in = mm < rows_m && d < a.dim;
              if (direct) {
                if (in) *reinterpret_cast<uint4*>(out) = v;
                out += RPI * a.dim;
                for (g += RPI; g >= a.group; g -= a.group) out += next_query;
              } else {
                if (in) *reinterpret_cast<uint4*>(part) = v;
                part += RPI * a.dim;
              }
            }
            __syncwarp();
          }
        }
        if (m < rows_m) {
          if (!ok) l = inv;
          if (!direct)
            (prefix ? a.prefix_ml : a.part_ml)[part_row + m] = make_float2(ref, l);
          else if (a.lse)
            a.lse[part_row + m] = l == 0.f ? INFINITY : ref + log2f(l);
        }
        tcgen05_before_sync();
      }
      // Over what attn_status_kernel wrote before, by whichever warp made its rows NaN.
      if (a.status && !prefix && t < it.mt && !ok && lane == 0) a.status[it.r] = SV_ST_TIMEOUT;
      if (t < it.mt && it.nt > 0) mbar_arrive(&sh.written[t]);
    }
  }
  __syncthreads();
  if (warp == 9) {
    tcgen05_after_sync();
    tmem_free512(tmem);
  }
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

// [rows][heads][slots][dim] with the given strides in elements; a box is 64 dimensions
// x 64 slots, zeros outside.  Dimensions of one entry, or whose entries coincide
// (stride 0), become dimensions of size one.
bool encode(CUtensorMap* map, const AttnArgs& a, const void* base, int64_t slots, int64_t heads, int64_t rows,
            int64_t s_slot, int64_t s_head, int64_t s_row) {
  const cuuint64_t dims[4] = {(cuuint64_t)a.dim, (cuuint64_t)slots, (cuuint64_t)(s_head ? heads : 1),
                              (cuuint64_t)(s_row ? rows : 1)};
  const cuuint64_t one = (cuuint64_t)a.dim * 2;
  const cuuint64_t strides[3] = {s_slot ? (cuuint64_t)s_slot * 2 : one, s_head ? (cuuint64_t)s_head * 2 : one,
                                 s_row ? (cuuint64_t)s_row * 2 : one};
  const cuuint32_t box[4] = {64, (cuuint32_t)BN, 1, 1}, steps[4] = {1, 1, 1, 1};
  return encode_fn()(map, a.dtype == 1 || a.halves ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                     const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DC, bool PAIRED, Source SRC>
cudaError_t tile(const AttnArgs& a, const Maps& maps, bool prefix, int tiles_m, cudaStream_t stream) {
  const int64_t rows_m = (int64_t)(prefix ? a.rows : 1) * a.n * a.group;
  const int64_t S = prefix ? a.p_splits : (a.o_splits ? a.o_splits : 1);
  const int64_t units = prefix ? a.kv_heads : (int64_t)a.rows * a.kv_heads;
  const int64_t items = (rows_m + tiles_m * BM - 1) / (tiles_m * BM) * S * units;
  if (items >= (int64_t)1 << 31 || (PAIRED && items > kSMs)) return cudaErrorInvalidValue;
  constexpr uint32_t bytes = Layout<DC, SRC>::kBytes;
  const cudaError_t e = allow_smem<attn_tile_kernel<T, DC, PAIRED, SRC>>(bytes);
  if (e != cudaSuccess) return e;
  attn_tile_kernel<T, DC, PAIRED, SRC><<<(unsigned)(items < kSMs ? items : kSMs), NT, bytes, stream>>>(
      a, maps, prefix, tiles_m, (int)units, (int)items);
  return cudaGetLastError();
}

template <typename T, Source SRC>
cudaError_t tile_any(const AttnArgs& a, const Maps& maps, bool prefix, const TileSplit& x, cudaStream_t stream) {
  if (a.dim <= 64)
    return x.paired ? tile<T, 1, true, SRC>(a, maps, prefix, 1, stream) : tile<T, 1, false, SRC>(a, maps, prefix, x.tiles, stream);
  if constexpr (SRC != kPairs) {
    if (x.paired) return tile<T, 2, true, SRC>(a, maps, prefix, 1, stream);
  }
  return tile<T, 2, false, SRC>(a, maps, prefix, x.tiles, stream);
}

}  // namespace

static std::atomic<int32_t> test_head{0};

cudaError_t launch_attn_tile(const AttnArgs& args, bool prefix, const TileSplit& split, cudaStream_t stream) {
  AttnArgs a = args;
  a.test_head = test_head.load(std::memory_order_relaxed) ? test_head.exchange(0) : 0;
  // A scale of zero weighs all slots alike; the least normal one does so without 0 * inf at the mask (kHalves: the
  // rows' factors are kept from zero instead).
  if (!(a.halves && a.dtype == 2) && fabsf(a.scale) < 0x1p-126f) a.scale = copysignf(0x1p-126f, a.scale);
  if (!encode_fn()) return cudaErrorNotSupported;
  Maps maps;
  memset(&maps, 0, sizeof maps);
  bool ok;
  if (prefix) {
    ok = encode(&maps.k, a, a.pk, a.prefix, a.kv_heads, 1, a.p_slot, a.p_head, 0) &&
         encode(&maps.v, a, a.pv, a.prefix, a.kv_heads, 1, a.p_slot, a.p_head, 0);
    maps.head_mul = a.p_head != 0;
  } else {
    ok = encode(&maps.k, a, a.k, a.capacity, a.kv_heads, a.rows, a.kv_slot, a.kv_head, a.kv_row) &&
         encode(&maps.v, a, a.v, a.capacity, a.kv_heads, a.rows, a.kv_slot, a.kv_head, a.kv_row);
    if (a.k_low)
      ok = ok && encode(&maps.low, a, a.k_low, a.capacity, a.kv_heads, a.rows, a.kv_slot, a.kv_head, a.kv_row);
    maps.head_mul = a.kv_head != 0;
    maps.row_mul = a.kv_row != 0;
  }
  if (!ok) return cudaErrorInvalidValue;
  if (a.halves)
    return a.dtype == 1 ? tile_any<__half, kPairs>(a, maps, prefix, split, stream)
                        : tile_any<__nv_bfloat16, kHalves>(a, maps, prefix, split, stream);
  return a.dtype == 1 ? tile_any<__half, kPlain>(a, maps, prefix, split, stream)
                      : tile_any<__nv_bfloat16, kPlain>(a, maps, prefix, split, stream);
}

}  // namespace sv

extern "C" void sv_test_attention_timeout(int32_t head) { sv::test_head = head + 1; }
