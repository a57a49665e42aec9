// sv_evict.cu -- eviction from the KV cache by accumulated attention weight.
//
// Per unit (layer, row, head) with n valid slots and a budget B < n, the B slots of
// largest rank stay: rank +inf for positions < sinks and for positions > newest -
// recent, else the slot's weight (NaN as -inf), ties to the lowest slot.  The
// survivors at slots >= B (in slot order) take the evicted slots below B (in slot
// order).  Sources and destinations are disjoint ranges, so the copies need no order
// among themselves, a repeated call gives the same result, and only the moved slots
// are read and written: 2 x 2 x moved x head_dim x element bytes per unit, plus 8
// bytes read and 8 written per slot of weights and positions.
//
// Selection is exact: the weights become ordered 32-bit keys, kept in shared memory,
// and the cut (the B-th largest key) is found by narrowing the interval between the
// smallest and the largest key of the unprotected slots, 1024 equal bins at a time: a
// count per bin, a scan from the top, the bin that holds the cut is the next interval.
// It ends when exactly B keys lie at or above a bin's edge (mostly in the second round)
// or the interval is one key (ties).  Fixed radix digits count worse: most weights share
// their leading digit, and additions to one bin wait for one another.  Halving the
// interval took twelve more rounds, each a barrier.  One bit per slot and prefix counts
// per 32-slot word then number the survivors and the holes, whose lists take the keys'
// place.  Several blocks share a unit when units are few: each selects for itself (the
// weights come from L2) and copies its part of the moves, which needs no exchange.
//
// Bound by the moved bytes when many slots move, by the selection's latency otherwise.
// Past kSmemKeys slots keys and positions are read again from global memory where they are
// needed and lists of moves are searched bit by bit.
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/starvector_sampling.h"
#include "sv_attention.h"

namespace {

constexpr int kBins = 1024;
constexpr int kSmemKeys = 24576;  // slots whose keys and positions are kept in shared memory
constexpr int kMostSlots = 1 << 20;
constexpr size_t kMostSmem = 220 * 1024;  // of a block's shared memory, for what depends on the capacity
// Words per count where counts for every word would not fit, from 600705 slots on.  (With counts
// for every eighth word 2 units of 40000 slots took 117 us, 105 with all, and 300 units of 30000
// slots 556 and 511; one of 600000 slots 905 and 1000.)
constexpr int kSparse = 4;
constexpr uint32_t kTop = 0xff800000u;  // the key of +inf, and of protected slots

struct EvictArgs {
  unsigned char* cache[2];
  int64_t s_layer, s_row, s_head, s_slot;  // bytes
  int dv;                                  // 16-byte vectors per slot and tensor
  int lanes_log2;                          // lanes that copy one slot (keys and values): at most 32
  int rows, heads, capacity, parts;
  const float* weights;  // [layers, rows, heads, capacity]
  const int32_t* positions;
  const int32_t* lengths;
  int budget, sinks, recent;
  float* weights_out;
  int32_t* positions_out;
  int32_t *lengths_out, *status;
};

__device__ __forceinline__ uint32_t ordered(float f) {
  const uint32_t u = __float_as_uint(f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ uint32_t rank_key(float w, int pos, int sinks, int recent_from) {
  if (pos < sinks || pos > recent_from) return kTop;
  if (w != w) return 0x007fffffu;  // -inf
  return ordered(w + 0.0f);        // -0 ties with +0
}

// The position of the k-th (from 0) set bit of words whose exclusive prefix counts, one
// for every WPC words, are `before` (n + 1 entries); word(i) gives the words.
template <int WPC, typename F>
__device__ __forceinline__ int select_bit(const int* before, int n, int k, F word) {
  int lo = 0, hi = n;  // before[lo] <= k < before[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (before[mid] <= k) lo = mid; else hi = mid;
  }
  int i = lo * WPC, left = k - before[lo];
  if (WPC > 1)
    for (int c; left >= (c = __popc(word(i))); ++i) left -= c;
  return i * 32 + (int)__fns(word(i), 0, left + 1);
}

// Four consecutive values from j on (fill past n); vec: the four can be read at once.
template <typename V, typename E> __device__ __forceinline__ void load4(const E* p, int j, int n, bool vec, E fill, E (&x)[4]) {
  if (vec) {
    const V v = *reinterpret_cast<const V*>(p + j);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (!vec) x[k] = j + k < n ? p[j + k] : fill;
    if (j + k >= n) x[k] = fill;
  }
}

// Bits of word i below / at and past slot B.
__device__ __forceinline__ uint32_t below_bits(int i, int B) {
  const int left = B - i * 32;
  return left >= 32 ? 0xffffffffu : (left <= 0 ? 0u : (1u << left) - 1u);
}

template <int NT, int PER_SM, bool SMEM_KEYS, int WPC>  // WPC: words per count
__global__ void __launch_bounds__(NT, PER_SM) kv_evict_kernel(const EvictArgs a) {
  constexpr int NW = NT / 32, PER = kBins / NT;  // bins per thread
  using Both = std::conditional_t<WPC == 1, uint32_t, unsigned long long>;  // two counts of a round in one value
  constexpr int kHalf = sizeof(Both) * 4;
  extern __shared__ uint32_t dyn[];
  __shared__ int bins[kBins];
  __shared__ int warp_count[NW], sh_bin, sh_over, sh_need;
  __shared__ int sh_newest;
  __shared__ Both warp_both[NW];
  __shared__ uint32_t round_ties[WPC == 1 ? 1 : NT / 8];
  __shared__ uint32_t sh_low, sh_high;
  const int unit = blockIdx.y, part = blockIdx.x;
  const int h = unit % a.heads, r = (unit / a.heads) % a.rows, layer = unit / (a.heads * a.rows);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int raw = a.lengths ? a.lengths[r] : a.capacity;
  const int n = min(max(raw, 0), a.capacity), B = a.budget;
  const int keep = min(n, B);
  const float* w = a.weights + (int64_t)unit * a.capacity;
  const int32_t* pos = a.positions + (int64_t)unit * a.capacity;
  float* wo = a.weights_out + (int64_t)unit * a.capacity;
  int32_t* po = a.positions_out + (int64_t)unit * a.capacity;
  if (layer == 0 && h == 0 && part == 0 && tid == 0) {
    if (a.lengths_out) a.lengths_out[r] = keep;
    if (a.status) a.status[r] = raw == n ? 0 : SV_ST_LENGTH;
  }
  // Weights and positions are read and written four slots at a time where units start
  // 16-byte aligned; each block writes the slots [slot0, slot1).
  const bool vec = !(a.capacity & 3) && !(((uintptr_t)a.weights | (uintptr_t)a.positions | (uintptr_t)a.weights_out |
                                           (uintptr_t)a.positions_out) & 15);
  const int per_part = ((a.capacity + a.parts - 1) / a.parts + 3) & ~3;
  const int slot0 = min(part * per_part, a.capacity), slot1 = min(slot0 + per_part, a.capacity);
  // Each slot's own weight and position go out as they are read; the moved follow at the end.
  auto write4 = [&](int j, const float (&x)[4], const int (&y)[4]) {
    if (vec) {
      *reinterpret_cast<float4*>(wo + j) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<int4*>(po + j) = make_int4(y[0], y[1], y[2], y[3]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (j + k < slot1) wo[j + k] = x[k], po[j + k] = y[k];
    }
  };
  auto copy_meta = [&](int from) {
#pragma unroll 2
    for (int j = max(slot0, from) + 4 * tid; j < slot1; j += 4 * NT) {
      float x[4];
      int y[4];
      load4<float4>(w, j, keep, vec, 0.f, x);
      load4<int4>(pos, j, keep, vec, -1, y);
      write4(j, x, y);
    }
  };
  if (n <= B) {
    copy_meta(0);
    return;
  }
  const int nw = (n + 31) >> 5, counts = (nw + WPC - 1) / WPC, n4 = (n + 3) & ~3;
  uint32_t* keys = dyn;                                    // [n4], later the lists of moves
  int* held = reinterpret_cast<int*>(keys + (SMEM_KEYS ? n4 : 0));  // [n4] positions
  uint32_t* kept = reinterpret_cast<uint32_t*>(held + (SMEM_KEYS ? n4 : 0));  // one bit per slot
  int* holes = reinterpret_cast<int*>(kept + nw);          // exclusive counts per WPC words, counts + 1
  int* comes = holes + counts + 1;

  // Newest position, then the keys and their range (protected ones left out).
  if (tid == 0) {
    sh_newest = INT32_MIN;
    sh_low = 0xffffffffu;
    sh_high = 0u;
  }
  int newest = INT32_MIN;
  if (SMEM_KEYS) {
#pragma unroll 2
    for (int j = 4 * tid; j < n; j += 4 * NT) {
      float x[4];
      int y[4];
      load4<float4>(w, j, n, vec, 0.f, x);
      load4<int4>(pos, j, n, vec, INT32_MIN, y);
      newest = max(max(max(newest, y[0]), max(y[1], y[2])), y[3]);
      *reinterpret_cast<float4*>(keys + j) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<int4*>(held + j) = make_int4(y[0], y[1], y[2], y[3]);
      if (j >= slot0 && j < slot1) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (j + k >= B) x[k] = 0.f, y[k] = -1;
        write4(j, x, y);
      }
    }
    copy_meta(n4);
  } else {
    for (int j = tid; j < n; j += NT) newest = max(newest, pos[j]);
    copy_meta(0);
  }
  newest = __reduce_max_sync(0xffffffffu, newest);
  __syncthreads();
  if (lane == 0) atomicMax(&sh_newest, newest);
  __syncthreads();
  // Positions above `from` are recent (none when recent is 0; all when that would lie below the type's range).
  const int64_t from64 = (int64_t)sh_newest - a.recent;
  const int from = (int)max(from64, (int64_t)INT32_MIN);
  const bool all_recent = from64 < INT32_MIN;
  auto make_key = [&](float x, int p) { return all_recent ? kTop : rank_key(x, p, a.sinks, from); };
  auto key = [&](int j) { return SMEM_KEYS ? keys[j] : make_key(w[j], pos[j]); };
  uint32_t low = 0xffffffffu, high = 0u;
  auto widen = [&](uint32_t k) {
    if (k < kTop) {
      low = min(low, k);
      high = max(high, k);
    }
  };
  if (SMEM_KEYS) {
    for (int j = 4 * tid; j < n; j += 4 * NT) {  // each thread's own four
      const float4 x = *reinterpret_cast<const float4*>(keys + j);
      const int4 y = *reinterpret_cast<const int4*>(held + j);
      uint4 k;
      k.x = make_key(x.x, y.x);
      widen(k.x);
      k.y = j + 1 < n ? make_key(x.y, y.y) : 0u;  // 0: below every slot's key
      if (j + 1 < n) widen(k.y);
      k.z = j + 2 < n ? make_key(x.z, y.z) : 0u;
      if (j + 2 < n) widen(k.z);
      k.w = j + 3 < n ? make_key(x.w, y.w) : 0u;
      if (j + 3 < n) widen(k.w);
      *reinterpret_cast<uint4*>(keys + j) = k;
    }
  } else {
    for (int j = tid; j < n; j += NT) widen(make_key(w[j], pos[j]));
  }
  low = __reduce_min_sync(0xffffffffu, low);
  high = __reduce_max_sync(0xffffffffu, high);
  if (lane == 0) {
    atomicMin(&sh_low, low);
    atomicMax(&sh_high, high);
  }
  __syncthreads();
  // cut, next: what lies at next and above stays (`above` slots), and of the slots in
  // [cut, next) all (exact) or, all being equal, the first `ties`.
  uint32_t cut = kTop, next = kTop + 1u;
  int above = 0;
  bool exact = false;
  if (sh_low <= sh_high) {  // some slot is not protected
    // Keys in [lo, hi]; above that, `over` ones (at first the protected, which bin kBins - 1 takes up).
    uint32_t lo = sh_low, hi = sh_high;
    int over = 0;
    for (bool first = true;; first = false) {
      // Bin width: the smallest power of two that covers the interval.
      const uint32_t span = hi - lo;
      const int shift = span < kBins ? 0 : 32 - __clz(span) - 10;
#pragma unroll
      for (int i = 0; i < PER; ++i) bins[tid + i * NT] = 0;
      int top = 0;
      __syncthreads();
      auto put = [&](uint32_t k) {
        top += k > hi;
        if (k >= lo && k <= hi) atomicAdd(&bins[(k - lo) >> shift], 1);
      };
      if (SMEM_KEYS) {
        for (int j = 4 * tid; j < n; j += 4 * NT) {
          const uint4 k = *reinterpret_cast<const uint4*>(keys + j);
          put(k.x), put(k.y), put(k.z), put(k.w);
        }
      } else {
        for (int j = tid; j < n; j += NT) put(key(j));
      }
      if (first) {
        top = __reduce_add_sync(0xffffffffu, top);
        if (lane == 0) warp_count[warp] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NW; ++i) over += warp_count[i];
      }
      __syncthreads();
      if (over >= B) break;  // the protected alone fill the budget: only in the first round
      // Scan from the top: thread x holds bins kBins - 1 - PER x and below.
      int c[PER], sum = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) sum += c[i] = bins[kBins - 1 - PER * tid - i];
      int upto = sum;
#pragma unroll
      for (int k = 1; k < 32; k <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, k);
        if (lane >= k) upto += x;
      }
      if (lane == 31) warp_count[warp] = upto;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NW; ++i)
        if (i < warp) upto += warp_count[i];
      int at = over + upto - sum;
      if (at < B && B <= at + sum) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          if (at < B && B <= at + c[i]) {
            sh_bin = kBins - 1 - PER * tid - i;
            sh_over = at;
            sh_need = c[i];
          }
          at += c[i];
        }
      }
      __syncthreads();
      const uint32_t edge = lo + ((uint32_t)sh_bin << shift);
      const int in_bin = sh_need;
      over = sh_over;
      if (over + in_bin == B || shift == 0) {
        exact = over + in_bin == B;
        cut = edge;
        next = exact ? hi : edge + 1u;
        above = over;
        break;
      }
      hi = min(hi, edge + (1u << shift) - 1u);
      lo = edge;
      __syncthreads();
    }
  }
  const int ties = B - above;

  // The first `ties` of the tied slots stay: warp 0 goes through the words of ties (of words
  // `first` on) in order.
  uint32_t* tie_words = WPC == 1 ? reinterpret_cast<uint32_t*>(holes) : round_ties;
  int tied = 0;
  auto take_ties = [&](int first, int words) {
    for (int i0 = 0; i0 < words && tied < ties; i0 += 32) {
      const int i = i0 + lane;
      uint32_t eq = i < words ? tie_words[i] : 0u, bits = 0u;
      const int c = __popc(eq);
      int s = c;
#pragma unroll
      for (int k = 1; k < 32; k <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, s, k);
        if (lane >= k) s += x;
      }
      int room = ties - (tied + s - c);
      tied += __shfl_sync(0xffffffffu, s, 31);
      if (room >= c) {
        bits = eq;
      } else {
        for (; room > 0; --room) {
          bits |= eq & (0u - eq);
          eq &= eq - 1u;
        }
      }
      if (i < words) kept[first + i] |= bits;
    }
  };
  // One bit per slot: a thread compares four, eight threads make a word.
  for (int i0 = 0; i0 < nw; i0 += NT / 8) {
    const int i = i0 + (tid >> 3), j = i * 32 + (tid & 7) * 4;
    uint32_t at = 0, over = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t k = j + e < n ? key(j + e) : 0u;
      at |= (uint32_t)(k >= cut) << e;
      over |= (uint32_t)(k >= next) << e;
    }
    at <<= (tid & 7) * 4;
    over <<= (tid & 7) * 4;
#pragma unroll
    for (int k = 1; k < 8; k <<= 1) {
      at |= __shfl_xor_sync(0xffffffffu, at, k);
      over |= __shfl_xor_sync(0xffffffffu, over, k);
    }
    if (!(tid & 7) && i < nw) {
      kept[i] = exact ? at : over;
      if (!exact) tie_words[WPC == 1 ? i : tid >> 3] = at & ~over;
    }
    if (WPC > 1 && !exact) {  // there is room for one round's ties only
      __syncthreads();
      if (warp == 0) take_ties(i0, min(NT / 8, nw - i0));
      __syncthreads();
    }
  }
  __syncthreads();
  if (WPC == 1 && !exact) {
    if (warp == 0) take_ties(0, nw);
    __syncthreads();
  }
  // Exclusive counts, those of WPC words per thread (both in one value: NT words hold at most
  // 32 NT = 2^15 slots, for sparse counts the value is wider).
  int nh = 0, nc = 0;
  for (int i0 = 0; i0 < counts; i0 += NT) {
    const int i = i0 + tid;
    Both c = 0;
#pragma unroll 1
    for (int k = 0; k < WPC; ++k) {
      const int x = i * WPC + k;
      const uint32_t bits = x < nw ? kept[x] : 0u, below = below_bits(x, B);
      if (x < nw) c += (Both)__popc(~bits & below) | (Both)__popc(bits & ~below) << kHalf;
    }
    Both s = c;
#pragma unroll
    for (int k = 1; k < 32; k <<= 1) {
      const Both x = __shfl_up_sync(0xffffffffu, s, k);
      if (lane >= k) s += x;
    }
    if (lane == 31) warp_both[warp] = s;
    __syncthreads();
    Both all = 0;
#pragma unroll
    for (int k = 0; k < NW; ++k) {
      if (k == warp) s += all;
      all += warp_both[k];
    }
    s -= c;
    constexpr Both low = ((Both)1 << kHalf) - 1;
    if (i < counts) {
      holes[i] = nh + (int)(s & low);
      comes[i] = nc + (int)(s >> kHalf);
    }
    nh += (int)(all & low);
    nc += (int)(all >> kHalf);
    __syncthreads();
  }
  if (tid == 0) holes[counts] = nh, comes[counts] = nc;
  __syncthreads();
  const int moved = comes[counts];
  auto hole_bits = [&](int i) { return ~kept[i] & below_bits(i, B); };
  auto come_bits = [&](int i) { return kept[i] & ~below_bits(i, B); };
  // The lists of survivors past the budget and of holes below it, over the keys (at most
  // n / 2 entries each).  Holes are few per word: a thread lists a word's.
  int *src_list = reinterpret_cast<int*>(keys), *dst_list = src_list + moved;
  if (SMEM_KEYS) {
    for (int i = tid; i < nw && i * 32 < B; i += NT) {
      int at = holes[i];
      for (uint32_t hb = hole_bits(i); hb; hb &= hb - 1u) dst_list[at++] = i * 32 + __ffs(hb) - 1;
    }
    for (int i = (B >> 5) + warp; i < nw; i += NW) {
      const uint32_t cb = come_bits(i);
      if (cb >> lane & 1u) src_list[comes[i] + __popc(cb & ((1u << lane) - 1u))] = i * 32 + lane;
    }
    __syncthreads();
  }
  auto src_of = [&](int k) { return SMEM_KEYS ? src_list[k] : select_bit<WPC>(comes, counts, k, come_bits); };
  auto dst_of = [&](int k) { return SMEM_KEYS ? dst_list[k] : select_bit<WPC>(holes, counts, k, hole_bits); };

  // Keys and values: a group of lanes per moved slot, four slots in flight.
  const int64_t base = layer * a.s_layer + r * a.s_row + h * a.s_head;
  const int vecs = a.cache[1] ? 2 * a.dv : a.dv, group = 1 << a.lanes_log2;
  const int groups = (a.parts * NT) >> a.lanes_log2, me = (part * NT + tid) >> a.lanes_log2;
  for (int e = tid & (group - 1); e < vecs; e += group) {
    unsigned char* cache = (e >= a.dv ? a.cache[1] + (e - a.dv) * 16 : a.cache[0] + e * 16) + base;
    for (int k0 = me; k0 < moved; k0 += 4 * groups) {
      uint4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (k0 + u * groups < moved)
          v[u] = *reinterpret_cast<const uint4*>(cache + src_of(k0 + u * groups) * a.s_slot);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (k0 + u * groups < moved) *reinterpret_cast<uint4*>(cache + dst_of(k0 + u * groups) * a.s_slot) = v[u];
    }
  }
  // Weights and positions of the moved (their places were written long ago by this block, barriers before).
  for (int k = tid; k < moved; k += NT) {
    const int dst = dst_of(k);
    if (dst < slot0 || dst >= slot1) continue;
    const int src = src_of(k);
    wo[dst] = w[src];
    po[dst] = SMEM_KEYS ? held[src] : pos[src];
  }
}

// Lengths updated in place: after the eviction, whose blocks all read them.
__global__ void __launch_bounds__(256) lengths_kernel(int32_t* lengths, int rows, int capacity, int budget) {
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r < rows) lengths[r] = min(min(max(lengths[r], 0), capacity), budget);
}

bool overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return a && b && x < y + (uintptr_t)b_bytes && y < x + (uintptr_t)a_bytes;
}

template <auto K> struct Kernel {
  static constexpr auto value = K;
};

}  // namespace

// See include/starvector_sampling.h.
extern "C" int sv_kv_evict(void* keys, void* values, int32_t elem_bytes, int32_t layers, int32_t rows, int32_t heads,
                           int32_t capacity, int32_t head_dim, int64_t stride_layer, int64_t stride_row,
                           int64_t stride_head, int64_t stride_slot, const float* weights, const int32_t* positions,
                           const int32_t* lengths, int32_t budget, int32_t sinks, int32_t recent, float* weights_out,
                           int32_t* positions_out, int32_t* lengths_out, int32_t* out_status, void* stream) {
  if (!keys || !weights || !positions || !weights_out || !positions_out) return SV_E_ARG;
  if (weights == weights_out || positions == positions_out) return SV_E_ARG;
  if (elem_bytes != 1 && elem_bytes != 2 && elem_bytes != 4) return SV_E_DTYPE;
  if (layers < 1 || rows < 1 || heads < 1 || capacity < 1 || head_dim < 1 || capacity > kMostSlots) return SV_E_SHAPE;
  if ((int64_t)layers * rows * heads > 65535) return SV_E_SHAPE;
  if (budget < 1 || budget > capacity || sinks < 0 || recent < 0 || (int64_t)sinks + recent > budget)
    return SV_E_RANGE;
  const int64_t row = (int64_t)head_dim * elem_bytes;
  const int64_t sb[4] = {stride_layer * elem_bytes, stride_row * elem_bytes, stride_head * elem_bytes,
                         stride_slot * elem_bytes};
  if (row > 16384) return SV_E_SHAPE;
  if (row % 16) return SV_E_ALIGN;
  for (int k = 0; k < 4; ++k)
    if (sb[k] % 16 || sb[k] < 0) return SV_E_ALIGN;
  if (reinterpret_cast<uintptr_t>(keys) % 16 || reinterpret_cast<uintptr_t>(values) % 16) return SV_E_ALIGN;
  // Every unit moves its own slots, in place.
  if (!sv::entries_apart<4>(row, {layers, rows, heads, capacity}, sb)) return SV_E_SHAPE;
  // Blocks read a row's length, weights and positions while others write: outputs lie apart
  // from the inputs and from one another (the new lengths may take the old ones' place).
  const bool in_place = lengths_out && lengths_out == lengths;
  const int64_t slots = 4ll * layers * rows * heads * capacity;
  const void* outs[4] = {weights_out, positions_out, out_status, lengths_out};
  const void* ins[3] = {weights, positions, lengths};
  for (int i = 0; i < 4; ++i) {
    const int64_t bytes = i < 2 ? slots : 4ll * rows;
    for (int k = 0; k < 3; ++k)
      if (!(in_place && i == 3 && k == 2) && overlap(outs[i], bytes, ins[k], k < 2 ? slots : 4ll * rows)) return SV_E_ARG;
    for (int k = 0; k < i; ++k)
      if (overlap(outs[i], bytes, outs[k], k < 2 ? slots : 4ll * rows)) return SV_E_ARG;
  }
  EvictArgs a;
  a.cache[0] = static_cast<unsigned char*>(keys);
  a.cache[1] = static_cast<unsigned char*>(values);
  a.s_layer = sb[0];
  a.s_row = sb[1];
  a.s_head = sb[2];
  a.s_slot = sb[3];
  a.dv = (int)(row / 16);
  a.rows = rows;
  a.heads = heads;
  a.capacity = capacity;
  a.weights = weights;
  a.positions = positions;
  a.lengths = lengths;
  a.budget = budget;
  a.sinks = sinks;
  a.recent = recent;
  a.weights_out = weights_out;
  a.positions_out = positions_out;
  a.lengths_out = in_place ? nullptr : lengths_out;
  a.status = out_status;
  const int units = layers * rows * heads;
  a.lanes_log2 = 0;
  while (a.lanes_log2 < 5 && (1 << a.lanes_log2) < (values ? 2 : 1) * a.dv) ++a.lanes_log2;
  // Many units: blocks of 256 threads, up to seven per SM (three to seven take the same time: 44.6-45.5 us
  // at 1024 units of about 2200 slots; at seven, 32 registers, a few words spill).  Few: one block of 1024 threads per SM in all, since each selects
  // anew (48 units of up to 8192 slots: 26 us, and 41 us with two rounds of such blocks).
  const bool many = units >= 296;
  a.parts = many || units > 148 ? 1 : 148 / units;
  if (a.parts > 16) a.parts = 16;
  const bool in_smem = capacity <= kSmemKeys;
  const size_t nw = (capacity + 31) / 32;
  const size_t dense = 4 * (3 * nw + 2 + (in_smem ? 2 * ((capacity + 3) & ~3) : 0));
  const bool sparse = dense > kMostSmem;
  const size_t smem = sparse ? 4 * (nw + 2 * ((nw + kSparse - 1) / kSparse + 1)) : dense;
  static_assert(4 * (3 * (kSmemKeys / 32) + 2 + 2 * kSmemKeys) <= kMostSmem, "the keys fit a block's shared memory");
  static_assert(4 * (kMostSlots / 32 + 2 * (kMostSlots / 32 / kSparse + 1)) <= kMostSmem, "bits and sparse counts fit");
  cudaError_t e;
  auto run = [&](auto which) {
    constexpr auto kernel = decltype(which)::value;
    e = smem > 40 * 1024 ? sv::allow_smem<kernel>(kMostSmem) : cudaSuccess;
    if (e != cudaSuccess) return;
    kernel<<<dim3(a.parts, units), many && !sparse ? 256 : 1024, smem, static_cast<cudaStream_t>(stream)>>>(a);
    e = cudaGetLastError();
  };
  if (sparse)
    run(Kernel<kv_evict_kernel<1024, 1, false, kSparse>>());
  else if (many)
    in_smem ? run(Kernel<kv_evict_kernel<256, 7, true, 1>>()) : run(Kernel<kv_evict_kernel<256, 7, false, 1>>());
  else
    in_smem ? run(Kernel<kv_evict_kernel<1024, 1, true, 1>>()) : run(Kernel<kv_evict_kernel<1024, 1, false, 1>>());
  if (in_place && e == cudaSuccess) {
    lengths_kernel<<<(rows + 255) / 256, 256, 0, static_cast<cudaStream_t>(stream)>>>(lengths_out, rows, capacity, budget);
    e = cudaGetLastError();
  }
  return e == cudaSuccess ? SV_OK : SV_E_CUDA;
}
