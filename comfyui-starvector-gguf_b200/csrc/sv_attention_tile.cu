// sv_attention_tile.cu -- attention of many query rows per key/value head (prompts,
// chunks of prompts, a batch over a shared prefix) on the fifth-generation tensor
// cores, float16 / bfloat16.
//
// A block holds up to two tiles of 128 query rows (row m = query i * G + head g of one
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
#include <cstring>
#include <type_traits>

#include "../../include/starvector_sampling.h"
#include "sv_attention.h"
#include "sv_tcgen05.cuh"

namespace sv {
namespace {

constexpr int NT = 384;
constexpr int BM = 128, BN = 64;
constexpr int RING = 4;            // steps (64 slots) whose keys and values are held
constexpr int STAGES = 2 * RING;
constexpr float kSlack = 8.f;
constexpr uint32_t kPoly = 0x22;  // which of eight pairs of weights take the polynomial
constexpr int kEdges = 16;  // tiles that not every row of a block sees whole: at most twelve, see whole()

template <int DC> struct Layout {
  static constexpr uint32_t kQHalf = BM * 128, kHalf = BN * 128;  // 64 dimensions of a tile's rows
  static constexpr uint32_t kQTile = DC * kQHalf, kTile = DC * kHalf;
  static constexpr uint32_t kRing = 2 * kQTile;                      // after two query tiles
  static constexpr uint32_t kBytes = kRing + STAGES * kTile + 1024;  // alignment slack
};

struct Shared {
  // full, ready: a stage's copy, and its edge-tile pass.  s_full, pv_done: a query tile's scores of step j and
  // its product of step j (they also free the step's keys and values); one barrier for each of the four steps
  // that the ring holds, so that none gets two phases ahead of who waits for it.
  uint64_t q_full[2], full[STAGES], ready[STAGES], s_full[2][RING], p_full[2][2], pv_done[2][RING], drained;
  uint32_t tmem;
  uint32_t bad[kEdges][BN / 32];  // per edge tile: its slots with values that are not finite
  int bad_from[kEdges], any_bad;
  volatile int abort;
};

struct Maps {
  CUtensorMap k, v;
  int32_t row_mul, head_mul;  // 0: all rows (heads) share one entry
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
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

// 2^x for two x at once on the FP32 pipes: x = n + f with n = round(x) (the addition of
// 1.5 2^23 leaves n in the low bits), 2^f by a polynomial of degree 4 (weighted least
// squares towards equal relative error on [-1/2, 1/2]: below 2.7e-6, under a 16-bit
// weight's rounding), n added to the exponent.  Below -126 it stays at 2^-126.
__device__ __forceinline__ void exp2_poly(uint64_t x2, float& u, float& v) {
  float x, y;
  unpack2(x2, x, y);
  x2 = pack2(fmaxf(x, -126.f), fmaxf(y, -126.f));
  const uint64_t big = pack2(12582912.f, 12582912.f), minus_big = pack2(-12582912.f, -12582912.f);
  const uint64_t t = add2(x2, big), n = add2(t, minus_big), f = fma2(n, pack2(-1.f, -1.f), x2);
  uint64_t p = fma2(pack2(0.00957010221f, 0.00957010221f), f, pack2(0.0559178628f, 0.0559178628f));
  p = fma2(p, f, pack2(0.240247443f, 0.240247443f));
  p = fma2(p, f, pack2(0.693121791f, 0.693121791f));
  p = fma2(p, f, pack2(0.999999285f, 0.999999285f));
  float tx, ty;
  unpack2(t, tx, ty);
  unpack2(p, x, y);
  u = __int_as_float(__float_as_int(x) + (__float_as_int(tx) << 23));
  v = __int_as_float(__float_as_int(y) + (__float_as_int(ty) << 23));
}

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

// A bounded wait that also ends when another role has given up.
__device__ __noinline__ bool wait_slow(Shared& sh, uint32_t bar, uint32_t phase) {
  const uint64_t t0 = gtimer_ns();
  for (;;) {
    if (mbar_try(bar, phase)) return true;
    if (sh.abort) return false;
    if (gtimer_ns() - t0 > 2000000000ull) {
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

template <typename T, int DC>
__global__ void __launch_bounds__(NT, 1) attn_tile_kernel(const __grid_constant__ AttnArgs a,
                                                          const __grid_constant__ Maps maps, const bool prefix,
                                                          const int tiles_m) {
  using L = Layout<DC>;
  extern __shared__ unsigned char dyn_raw[];
  __shared__ Shared sh;
  unsigned char* dyn = dyn_raw + ((1024u - (smem_u32(dyn_raw) & 1023u)) & 1023u);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nG = a.n * a.group;
  const int rows_m = prefix ? a.rows * nG : nG;
  const int S = prefix ? a.p_splits : max(a.o_splits, 1);
  // The last rows see the most slots under a causal mask: they start first.
  const int blocks_m = gridDim.x / S;
  const int split = blockIdx.x % S, m0 = (blocks_m - 1 - blockIdx.x / S) * tiles_m * BM;
  const int unit = blockIdx.y;
  const int h = prefix ? unit : unit % a.kv_heads, r_own = prefix ? 0 : unit / a.kv_heads;
  const int mt = min(tiles_m, (rows_m - m0 + BM - 1) / BM);  // query tiles that hold rows

  // Slots: [a0, a1) sinks before the window, [b0, b1) the rest.
  RowSpan sp = {0, a.prefix};
  int a0 = 0, a1 = 0, b0 = 0, b1 = a.prefix;
  const int m_last = min(m0 + tiles_m * BM, rows_m) - 1;
  if (!prefix) {
    sp = row_span(a, r_own);
    const int pf = sp.end - a.n + m0 / a.group, pl = sp.end - a.n + m_last / a.group;
    b0 = window_low(a, sp.start, pf);
    b1 = pl < sp.start ? b0 : max(pl + 1, b0);
    a0 = sp.start;
    a1 = pl >= sp.start ? max(a0, min(sp.start + a.sinks, b0)) : a0;
  }
  const int ta = (a1 - a0 + BN - 1) / BN, tiles = ta + (b1 - b0 + BN - 1) / BN;
  const int t0 = (int)((int64_t)tiles * split / S), nt = (int)((int64_t)tiles * (split + 1) / S) - t0;
  auto tile_at = [&](int j, int& j0, int& jend) {
    const int t = t0 + j;
    j0 = t < ta ? a0 + t * BN : b0 + (t - ta) * BN;
    jend = t < ta ? a1 : b1;
  };
  // Whether rows that all see the slots [from, to] of the window see the whole tile.
  auto whole = [&](int j, int from, int to) {
    int j0, jend;
    tile_at(j, j0, jend);
    if (j0 + BN > jend) return false;
    return prefix || t0 + j < ta || (j0 >= from && j0 + BN - 1 <= to);
  };
  auto seen_by_all = [&](int first, int last, int& from, int& to) {  // rows [first, last]
    from = window_low(a, sp.start, sp.end - a.n + last / a.group);
    to = sp.end - a.n + first / a.group;
  };

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.q_full[i], 128);
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
    mbar_init(&sh.drained, 2);
    sh.any_bad = 0;
    for (int i = 0; i < kEdges; ++i)
      for (int k = 0; k < BN / 32; ++k) sh.bad[i][k] = 0;
    sh.abort = 0;
    mbar_init_fence();
  }
  if (warp == 9) tmem_alloc512(&sh.tmem);
  tcgen05_before_sync();
  __syncthreads();
  tcgen05_after_sync();
  const uint32_t tmem = sh.tmem;

  if (warp == 8) {
    // ------------------------------------------------------------- copies
    if (lane == 0 && nt > 0) {
      tma_prefetch_map(&maps.k);
      tma_prefetch_map(&maps.v);
      int issued = 0;
      for (; issued < 2 * nt; ++issued) {
        const int st = issued % STAGES, step = (issued >> 1) % RING;
        bool free = true;  // once both tiles' products of four steps ago are done
        for (int t = 0; t < mt && issued >= STAGES; ++t)
          free = free && wait_one(sh, issued & 1 ? &sh.pv_done[t][step] : &sh.s_full[t][step], (issued / STAGES - 1) & 1);
        if (!free) break;
        int j0, jend;
        tile_at(issued >> 1, j0, jend);
        mbar_expect_tx(&sh.full[st], L::kTile);
        const CUtensorMap* map = issued & 1 ? &maps.v : &maps.k;
#pragma unroll
        for (int d = 0; d < DC; ++d)
          tma_load4(dyn + L::kRing + st * L::kTile + d * L::kHalf, map, d * 64, j0, h * maps.head_mul,
                    r_own * maps.row_mul, &sh.full[st]);
      }
      // After an abort nothing may still be landing when the block ends.
      if (sh.abort)
        for (int i = max(0, issued - STAGES); i < issued; ++i)
          mbar_wait(&sh.full[i % STAGES], (i / STAGES) & 1);
    }
  } else if (warp == 9 || warp == 10) {
    // ------------------------------------------------------------- products
    constexpr uint32_t wqk = mma_word(Half16<T>::bf16, BN, false), wpv = mma_word(Half16<T>::bf16, 64 * DC, true);
    // Descriptors are sums of a base and constants, so that they stay in uniform registers.
    const uint64_t q_desc = smem_desc(smem_u32(dyn), 16), k_desc = smem_desc(smem_u32(dyn) + L::kRing, 16),
                   v_desc = smem_desc(smem_u32(dyn) + L::kRing, L::kHalf);
    constexpr uint32_t kStep = L::kTile >> 4;
    const bool leader = elect_one();
    constexpr uint32_t kQStep = L::kQTile >> 4;
    // Loop bounds and addresses that the compiler can tell are the same in all lanes (a
    // reduction's result is), or every product would first move its operands to uniform
    // registers: about 50 cycles each.
    const int steps = __reduce_max_sync(0xffffffffu, nt);
    const uint32_t tm = __reduce_max_sync(0xffffffffu, tmem);
    // One lane waits and issues.  After an abort its waits fail at once and the rest of the
    // loop computes on what is there, which nobody uses.
    const int t = warp - 9;
    const uint32_t s_at = tm + t * 128, o_at = tm + 256 + t * 128;
    const uint64_t qd = q_desc + t * kQStep;
    auto qk = [&](int j) {
      const uint64_t kd = k_desc + (2 * j) % STAGES * kStep;
#pragma unroll
      for (int k = 0; k < 4 * DC; ++k)
        mma_ss(s_at + (j & 1) * BN, qd + (((k >> 2) * L::kQHalf + (k & 3) * 32) >> 4),
               kd + (((k >> 2) * L::kHalf + (k & 3) * 32) >> 4), wqk, k != 0);
      mma_commit(&sh.s_full[t][j % RING]);
    };
    if (leader && t < mt && steps > 0) {
      wait_one(sh, &sh.q_full[t], 0);
      for (int j = 0; j < min(steps, 2); ++j) {
        wait_one(sh, &sh.full[2 * j], 0);
        qk(j);
      }
    }
    __syncwarp();
    if (t < mt) {
#pragma unroll 1
      for (int j = 0; j < steps; ++j) {
        const int vi = 2 * j + 1, ki = 2 * j + 4;
        if (leader) {
          wait_one(sh, &sh.ready[vi % STAGES], (vi / STAGES) & 1);
          wait_one(sh, &sh.p_full[t][j & 1], (j >> 1) & 1);
          tcgen05_after_sync();
          const uint64_t vd = v_desc + (vi % STAGES) * kStep;
#pragma unroll
          for (int k = 0; k < BN / 16; ++k)
            mma_ts(o_at, s_at + (j & 1) * BN + k * 8, vd + k * (2048 >> 4), wpv, j != 0 || k != 0);
          mma_commit(&sh.pv_done[t][j % RING]);
          if (j + 2 < steps) {
            wait_one(sh, &sh.full[ki % STAGES], (ki / STAGES) & 1);
            qk(j + 2);
          }
        }
        __syncwarp();
      }
    }
    if (__any_sync(0xffffffffu, sh.abort)) {  // the products in flight
      if (leader) {
        mma_commit(&sh.drained);
        mbar_wait(&sh.drained, 0);
      }
      __syncwarp();
    }
  } else if (warp == 11) {
    // ------------------------------------------------------------- values of edge tiles
    int edge = 0, from, to;
    seen_by_all(m0, m_last, from, to);
    for (int j = 0; j < nt; ++j) {
      const int vi = 2 * j + 1, st = vi % STAGES;
      if (!wait(sh, &sh.full[st], (vi / STAGES) & 1)) break;
      if (!whole(j, from, to)) {
        int j0, jend;
        tile_at(j, j0, jend);
        unsigned char* vb = dyn + L::kRing + st * L::kTile;
        // A vector of 16 bytes at a time; the swizzle permutes vectors within a row only.
        for (int x = lane; x < BN * DC * 8; x += 32) {
          const int half = x / (BN * 8), row = (x >> 3) & (BN - 1), vec = x & 7;
          uint4* p = reinterpret_cast<uint4*>(vb + half * L::kHalf + row * 128 + vec * 16);
          if (j0 + row >= jend) {
            *p = make_uint4(0u, 0u, 0u, 0u);
            continue;
          }
          uint4 v = *p;
          uint32_t* w = reinterpret_cast<uint32_t*>(&v);
          bool bad = false;
          constexpr uint32_t E = Half16<T>::expo;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if ((w[k] & E) == E) w[k] &= 0xffff0000u, bad = true;
            if ((w[k] & (E << 16)) == E << 16) w[k] &= 0xffffu, bad = true;
          }
          if (bad) {
            *p = v;
            atomicOr(&sh.bad[edge][row >> 5], 1u << (row & 31));
            sh.bad_from[edge] = j0;
            sh.any_bad = 1;
          }
        }
        fence_proxy_async_smem();
        edge = min(edge + 1, kEdges - 1);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.ready[st]);
    }
  } else {
    // ------------------------------------------------------------- softmax and output
    const int t = warp >> 2, row = tid & 127;
    if (t < mt) {
      const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;  // a negative scale turns the queries' signs
      const float scale = fabsf(a.scale);
      const int mfirst = m0 + t * BM, mlast = min(mfirst + BM, rows_m) - 1;
      const int m = mfirst + row;
      const int r = prefix ? m / nG : r_own, mr = prefix ? m - r * nG : m;
      const int i = mr / a.group, g = mr - i * a.group;
      {  // a thread brings its own row: all its vectors in flight at once
        uint4 v[DC * 8];
        const T* src = static_cast<const T*>(a.q) + r * a.q_row + i * a.q_tok + (int64_t)(h * a.group + g) * a.q_head;
#pragma unroll
        for (int c = 0; c < DC * 8; ++c)
          v[c] = m < rows_m && c * 8 < a.dim ? __ldg(reinterpret_cast<const uint4*>(src) + c) : make_uint4(0u, 0u, 0u, 0u);
        unsigned char* qb = dyn + t * L::kQTile + row * 128;
#pragma unroll
        for (int c = 0; c < DC * 8; ++c) {
          v[c].x ^= flip, v[c].y ^= flip, v[c].z ^= flip, v[c].w ^= flip;
          *reinterpret_cast<uint4*>(qb + (c >> 3) * L::kQHalf + (((c & 7) ^ (row & 7)) << 4)) = v[c];
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(&sh.q_full[t]);

      const int pos = prefix ? a.prefix : sp.end - a.n + i;
      const int low = prefix ? 0 : window_low(a, sp.start, pos);
      const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);
      const uint32_t o_at = lanes + 256 + t * 128;
      int from, to;
      seen_by_all(mfirst, mlast, from, to);
      auto products_done = [&](int j) { return wait(sh, &sh.pv_done[t][j % RING], (j / RING) & 1); };
      float ref = -INFINITY, l = 0.f;
      bool ok = true;
      for (int j = 0; j < nt; ++j) {
        ok = wait(sh, &sh.s_full[t][j % RING], (j / RING) & 1);
        if (!ok) break;
        tcgen05_after_sync();
        const uint32_t s_at = lanes + t * 128 + (j & 1) * BN;
        float s[BN];
        tmem_load64(s_at, s);
        const bool all_seen = whole(j, from, to);
        if (!all_seen) {
          int j0, jend;
          tile_at(j, j0, jend);
          const int r1 = min(pos + 1, jend) - j0, r0 = low - j0, s1 = min(sp.start + a.sinks, min(pos + 1, jend)) - j0;
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
        const bool need = !(top <= ref + kSlack) && top != -INFINITY;
        if (__any_sync(0xffffffffu, need)) {
          const float f = need ? ex2(ref - top) : 1.f;
          if (need) ref = top;
          l *= f;
          if (j > 0) {  // the product before must be in, and this tile's waits for these weights
            ok = products_done(j - 1);
            if (!ok) break;
            tcgen05_after_sync();
#pragma unroll 1
            for (int c = 0; c < 64 * DC; c += 32) {
              float o[32];
              tmem_load32(o_at + c, o);
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] *= f;
              tmem_store32(o_at + c, o);
            }
          }
        }
        // Nothing seen yet: weights of zero; a maximum of +inf: NaN, as inf - inf.
        const float at = ref == -INFINITY ? 0.f : (ref == INFINITY ? __int_as_float(0x7fc00000) : ref);
        const uint64_t scale2 = pack2(scale, scale), at2 = pack2(-at, -at);
        uint64_t sum[2] = {0, 0};
        // The special function unit takes 8 cycles for a warp's 32 exponentials: in tiles
        // without hidden slots some go to the FP32 pipes instead.
        auto weights = [&](auto mixed) {
          {
            uint32_t p[32];
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              float x, y;
              const uint64_t z = fma2(pack2(s[2 * k], s[2 * k + 1]), scale2, at2);
              if (decltype(mixed)::value && kPoly >> (k & 7) & 1) {
                exp2_poly(z, x, y);
              } else {
                unpack2(z, x, y);
                x = ex2(x);
                y = ex2(y);
              }
              sum[k & 1] = add2(sum[k & 1], pack2(x, y));
              p[k] = Half16<T>::pack(x, y);
            }
            tmem_store32(s_at, p);
          }
        };
        if (all_seen)
          weights(std::true_type());
        else
          weights(std::false_type());
        float sx, sy;
        unpack2(add2(sum[0], sum[1]), sx, sy);
        l += sx + sy;
        tmem_wait_store();
        tcgen05_before_sync();
        mbar_arrive(&sh.p_full[t][j & 1]);
      }
      if (ok && nt > 0) {
        ok = products_done(nt - 1);
        tcgen05_after_sync();
      }
      ok = __all_sync(0xffffffffu, ok && !sh.abort);
      const bool any_bad = *static_cast<volatile int*>(&sh.any_bad) != 0;
      const bool direct = !prefix && a.o_splits == 0;
      const int64_t idx = ((int64_t)r * a.kv_heads + h) * nG + mr;
      const float inv = !ok ? __int_as_float(0x7fc00000) : (l == 0.f ? 0.f : (direct ? 1.f / l : 1.f));
      const int64_t all = (int64_t)a.rows * a.kv_heads * nG;
#pragma unroll 1
      for (int c = 0; c < 64 * DC; c += 32) {
        float o[32];
        if (ok && nt > 0) {
          tmem_load32(o_at + c, o);
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = 0.f;
        }
        if (m < rows_m) {
        if (any_bad) {  // values that are not finite, for the rows that see them
          for (int e = 0; e < kEdges * BN; ++e) {
            if (!(sh.bad[e / BN][(e % BN) >> 5] >> (e & 31) & 1u)) continue;
            const int slot = sh.bad_from[e / BN] + e % BN;
            if (!prefix && !slot_seen(a, sp.start, pos, low, slot)) continue;
            const T* vp = static_cast<const T*>(prefix ? a.pv : a.v) +
                          (prefix ? h * a.p_head + slot * a.p_slot
                                  : r_own * a.kv_row + h * a.kv_head + slot * a.kv_slot);
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
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] *= inv;
        if (direct) {
          T* out = static_cast<T*>(a.out) + (((int64_t)r * a.n + i) * a.heads + h * a.group + g) * a.dim;
#pragma unroll
          for (int k = 0; k < 32; k += 8)
            if (c + k < a.dim)
              *reinterpret_cast<uint4*>(out + c + k) =
                  make_uint4(Half16<T>::pack(o[k], o[k + 1]), Half16<T>::pack(o[k + 2], o[k + 3]),
                             Half16<T>::pack(o[k + 4], o[k + 5]), Half16<T>::pack(o[k + 6], o[k + 7]));
        } else {
          float* out = (prefix ? a.prefix_o : a.part_o) + ((int64_t)split * all + idx) * a.dim;
#pragma unroll
          for (int k = 0; k < 32; k += 4)
            if (c + k < a.dim)
              *reinterpret_cast<float4*>(out + c + k) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
        }
        }
        __syncwarp();
      }
      if (m < rows_m) {
        if (!ok) l = inv;
        if (!direct)
          (prefix ? a.prefix_ml : a.part_ml)[(int64_t)split * all + idx] = make_float2(ref, l);
        else if (a.lse)
          a.lse[idx] = l == 0.f ? INFINITY : ref + log2f(l);
      }
      tcgen05_before_sync();
    }
  }
  __syncthreads();
  if (warp == 9) {
    tcgen05_after_sync();
    tmem_free512(tmem);
  }
  if (a.status && !prefix && tid == 0 && h == 0) {
    const int e = a.lengths ? a.lengths[r_own] : a.capacity, s = a.starts ? a.starts[r_own] : 0;
    if (sh.abort)
      a.status[r_own] = SV_ST_TIMEOUT;
    else if (blockIdx.x == 0)
      a.status[r_own] = (e < 0 || e > a.capacity || s < 0 || s > max(e, 0)) ? SV_ST_LENGTH : 0;
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
  return encode_fn()(map, a.dtype == 1 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                     const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DC>
cudaError_t tile(const AttnArgs& a, const Maps& maps, bool prefix, int tiles_m, cudaStream_t stream) {
  const int64_t rows_m = (int64_t)(prefix ? a.rows : 1) * a.n * a.group;
  const int64_t S = prefix ? a.p_splits : (a.o_splits ? a.o_splits : 1);
  const dim3 grid((unsigned)((rows_m + tiles_m * BM - 1) / (tiles_m * BM) * S),
                  (unsigned)(prefix ? a.kv_heads : a.rows * a.kv_heads));
  const cudaError_t e = allow_smem<attn_tile_kernel<T, DC>>(Layout<DC>::kBytes);
  if (e != cudaSuccess) return e;
  attn_tile_kernel<T, DC><<<grid, NT, Layout<DC>::kBytes, stream>>>(a, maps, prefix, tiles_m);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_attn_tile(const AttnArgs& args, bool prefix, int tiles_m, cudaStream_t stream) {
  AttnArgs a = args;
  // A scale of zero weighs all slots alike; a tiny one does so without 0 * inf at the mask.
  if (fabsf(a.scale) < 1e-30f) a.scale = 1e-30f;
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
    maps.head_mul = a.kv_head != 0;
    maps.row_mul = a.kv_row != 0;
  }
  if (!ok) return cudaErrorInvalidValue;
  if (a.dtype == 1)
    return a.dim <= 64 ? tile<__half, 1>(a, maps, prefix, tiles_m, stream)
                       : tile<__half, 2>(a, maps, prefix, tiles_m, stream);
  return a.dim <= 64 ? tile<__nv_bfloat16, 1>(a, maps, prefix, tiles_m, stream)
                     : tile<__nv_bfloat16, 2>(a, maps, prefix, tiles_m, stream);
}

}  // namespace sv
