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
// Selection is an exact radix select of the B-th largest 32-bit ordered key (four
// passes of 8 bits over keys kept in shared memory), then one bit per slot and prefix
// counts per 32-slot word: the k-th survivor and the k-th hole are found by a binary
// search over the counts, so no list is built.  Several blocks share a unit: each
// selects for itself (the weights are read from L2) and copies its part of the moves,
// which needs no exchange between blocks.
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/starvector_sampling.h"

namespace {

constexpr int NT = 512;
constexpr int NW = NT / 32;
constexpr int kSmemKeys = 32768;  // slots whose keys are kept in shared memory

struct EvictArgs {
  unsigned char* cache[2];
  int64_t s_layer, s_row, s_head, s_slot;  // bytes
  int dv;                                  // 16-byte vectors per slot
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

__device__ __forceinline__ uint32_t rank_key(float w, int pos, int sinks, int64_t recent_from) {
  if (pos < sinks || pos >= recent_from) return 0xff800000u;  // +inf
  if (w != w) return 0x007fffffu;                             // -inf
  return ordered(w + 0.0f);                                   // -0 ties with +0
}

// The position of the k-th (from 0) set bit of the words whose exclusive prefix counts
// are `before` (nw + 1 entries); word(i) gives the words.
template <typename F>
__device__ __forceinline__ int select_bit(const int* before, int nw, int k, F word) {
  int lo = 0, hi = nw;  // before[lo] <= k < before[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (before[mid] <= k) lo = mid; else hi = mid;
  }
  return lo * 32 + (int)__fns(word(lo), 0, k - before[lo] + 1);
}

template <bool SMEM_KEYS>
__global__ void __launch_bounds__(NT) kv_evict_kernel(const EvictArgs a) {
  extern __shared__ uint32_t dyn[];
  __shared__ uint32_t hist[256];
  __shared__ int warp_sum[2][NW];
  __shared__ int sh_newest, sh_need, carry[2];
  __shared__ uint32_t sh_prefix;
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
  if (n <= B) {
    for (int j = part * NT + tid; j < a.capacity; j += a.parts * NT) {
      wo[j] = j < n ? w[j] : 0.f;
      po[j] = j < n ? pos[j] : -1;
    }
    return;
  }
  const int nw = (n + 31) >> 5;
  uint32_t* kept = dyn;                                    // one bit per slot
  int* holes = reinterpret_cast<int*>(kept + nw);          // exclusive counts per word, nw + 1
  int* comes = holes + nw + 1;
  uint32_t* keys = reinterpret_cast<uint32_t*>(comes + nw + 1);

  // Newest position, then the ranks.
  int newest = INT32_MIN;
  for (int j = tid; j < n; j += NT) newest = max(newest, pos[j]);
  newest = __reduce_max_sync(0xffffffffu, newest);
  if (tid == 0) sh_newest = INT32_MIN;
  __syncthreads();
  if (lane == 0) atomicMax(&sh_newest, newest);
  __syncthreads();
  const int64_t from = (int64_t)sh_newest - a.recent + 1;
  if (SMEM_KEYS)
    for (int j = tid; j < n; j += NT) keys[j] = rank_key(w[j], pos[j], a.sinks, from);
  auto key = [&](int j) { return SMEM_KEYS ? keys[j] : rank_key(w[j], pos[j], a.sinks, from); };

  // Radix select of the B-th largest key.
  if (tid == 0) {
    sh_prefix = 0;
    sh_need = B;
  }
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += NT) hist[i] = 0;
    __syncthreads();
    const uint32_t prefix = sh_prefix;
    const uint32_t high = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
    for (int j = tid; j < n; j += NT) {
      const uint32_t k = key(j);
      if ((k & high) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (warp == 0) {
      // Lane l holds bins 255 - 8 l down to 248 - 8 l.
      int c[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += c[i] = (int)hist[255 - 8 * lane - i];
      int incl = sum;
#pragma unroll
      for (int k = 1; k < 32; k <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, incl, k);
        if (lane >= k) incl += x;
      }
      const int need = sh_need;
      int above = incl - sum;
      if (above < need && need <= incl) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (above < need && need <= above + c[i]) {
            sh_prefix = prefix | ((uint32_t)(255 - 8 * lane - i) << shift);
            sh_need = need - above;
            above = need;  // found
          } else {
            above += c[i];
          }
        }
      }
    }
    __syncthreads();
  }
  const uint32_t cut = sh_prefix;
  const int ties = sh_need;  // of the slots at the cut, the first `ties` stay

  // One bit per slot and the prefix counts, 32 x NW slots at a time.
  if (tid == 0) carry[0] = carry[1] = 0;
  int tie_base = 0;
  for (int w0 = 0; w0 < nw; w0 += NW) {
    const int word = w0 + warp, j = word * 32 + lane;
    const uint32_t k = j < n ? key(j) : 0u;
    const unsigned eq = __ballot_sync(0xffffffffu, j < n && k == cut);
    const unsigned gt = __ballot_sync(0xffffffffu, j < n && k > cut);
    if (lane == 0) warp_sum[0][warp] = __popc(eq);
    __syncthreads();
    int before = tie_base, all = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      const int c = warp_sum[0][i];
      if (i < warp) before += c;
      all += c;
    }
    tie_base += all;
    const bool stays = (gt >> lane & 1u) ||
                       ((eq >> lane & 1u) && before + __popc(eq & ((1u << lane) - 1u)) < ties);
    const unsigned bits = __ballot_sync(0xffffffffu, stays);
    if (lane == 0 && word < nw) kept[word] = bits;
    __syncthreads();
  }
  auto hole_bits = [&](int i) {
    const int left = B - i * 32;
    const uint32_t below = left >= 32 ? 0xffffffffu : (left <= 0 ? 0u : (1u << left) - 1u);
    return ~kept[i] & below;
  };
  auto come_bits = [&](int i) {
    const int left = B - i * 32;
    const uint32_t below = left >= 32 ? 0xffffffffu : (left <= 0 ? 0u : (1u << left) - 1u);
    return kept[i] & ~below;
  };
  for (int w0 = 0; w0 < nw; w0 += NT) {
    const int i = w0 + tid;
    const int c0 = i < nw ? __popc(hole_bits(i)) : 0, c1 = i < nw ? __popc(come_bits(i)) : 0;
    int s0 = c0, s1 = c1;
#pragma unroll
    for (int k = 1; k < 32; k <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, s0, k), y = __shfl_up_sync(0xffffffffu, s1, k);
      if (lane >= k) s0 += x, s1 += y;
    }
    if (lane == 31) warp_sum[0][warp] = s0, warp_sum[1][warp] = s1;
    __syncthreads();
    int b0 = carry[0], b1 = carry[1];
    for (int k = 0; k < warp; ++k) b0 += warp_sum[0][k], b1 += warp_sum[1][k];
    if (i < nw) holes[i] = b0 + s0 - c0, comes[i] = b1 + s1 - c1;
    __syncthreads();
    if (tid == NT - 1) carry[0] = b0 + s0, carry[1] = b1 + s1;
    __syncthreads();
  }
  if (tid == 0) holes[nw] = carry[0], comes[nw] = carry[1];
  __syncthreads();
  const int moved = comes[nw];

  // Weights and positions.
  for (int j = part * NT + tid; j < a.capacity; j += a.parts * NT) {
    float x = 0.f;
    int p = -1;
    if (j < B) {
      int from_slot = j;
      const uint32_t hb = hole_bits(j >> 5);
      if (hb >> (j & 31) & 1u)
        from_slot = select_bit(comes, nw, holes[j >> 5] + __popc(hb & ((1u << (j & 31)) - 1u)), come_bits);
      x = w[from_slot];
      p = pos[from_slot];
    }
    wo[j] = x;
    po[j] = p;
  }
  // Keys and values: one warp per moved slot.
  const int64_t base = layer * a.s_layer + r * a.s_row + h * a.s_head;
  for (int k = part * NW + warp; k < moved; k += a.parts * NW) {
    const int64_t src = base + select_bit(comes, nw, k, come_bits) * a.s_slot;
    const int64_t dst = base + select_bit(holes, nw, k, hole_bits) * a.s_slot;
    for (int x = lane; x < 2 * a.dv; x += 32) {
      const int c = x >= a.dv, v = c ? x - a.dv : x;
      if (a.cache[c])
        *reinterpret_cast<uint4*>(a.cache[c] + dst + v * 16) =
            *reinterpret_cast<const uint4*>(a.cache[c] + src + v * 16);
    }
  }
}

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
  if (layers < 1 || rows < 1 || heads < 1 || capacity < 1 || head_dim < 1 || capacity > (1 << 20)) return SV_E_SHAPE;
  if ((int64_t)layers * rows * heads > 65535) return SV_E_SHAPE;
  if (budget < 1 || budget > capacity || sinks < 0 || recent < 0 || (int64_t)sinks + recent > budget)
    return SV_E_RANGE;
  const int64_t row = (int64_t)head_dim * elem_bytes;
  const int64_t sb[4] = {stride_layer * elem_bytes, stride_row * elem_bytes, stride_head * elem_bytes,
                         stride_slot * elem_bytes};
  if (row % 16) return SV_E_ALIGN;
  for (int k = 0; k < 4; ++k)
    if (sb[k] % 16 || sb[k] < 0) return SV_E_ALIGN;
  if (reinterpret_cast<uintptr_t>(keys) % 16 || reinterpret_cast<uintptr_t>(values) % 16) return SV_E_ALIGN;
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
  a.lengths_out = lengths_out;
  a.status = out_status;
  const int units = layers * rows * heads;
  a.parts = units >= 592 ? 1 : (592 + units - 1) / units;
  if (a.parts > 16) a.parts = 16;
  const bool in_smem = capacity <= kSmemKeys;
  const size_t nw = (capacity + 31) / 32;
  const size_t smem = 4 * (3 * nw + 2 + (in_smem ? capacity : 0));
  auto kernel = in_smem ? kv_evict_kernel<true> : kv_evict_kernel<false>;
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return SV_E_CUDA;
  kernel<<<dim3(a.parts, units), NT, smem, static_cast<cudaStream_t>(stream)>>>(a);
  return cudaGetLastError() == cudaSuccess ? SV_OK : SV_E_CUDA;
}
