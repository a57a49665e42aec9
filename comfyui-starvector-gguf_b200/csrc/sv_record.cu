// sv_record.cu -- the cache held in 4 bits (sv_record.cuh): writing and reading records.
//
// A group of threads takes one slot of one head: thread (i, y) of it block i's dimensions
// 8 y .. 8 y + 7 and 16 + 8 y .. 16 + 8 y + 7, which are the words t = 2 y and 2 y + 1 of the
// block.  Both kernels move each byte once; a warp's loads and stores cover whole
// sectors.  Reading is bound by memory (8 x 4096 slots of four heads of 128 in bfloat16: 16 us, floor 13.4; four
// slots a thread where there are many, 19.5 us with one).  Writing is bound by its instructions (8192 tokens of four heads
// in 9.3 us; one slot a thread: with four a call under a profiler took 17.5 us, 14.7 with one).
//
// Writing.  Of a group's finite values x, clamped to +-32768, with extremes lo, hi:
//   scale = f16((hi - lo) / 15),  mid = f16(lo + 8 scale),
//   c = 8 + the whole number next to (x - mid) / scale (ties to the even one), within 0..15,
// each rounded once from the exact number.  In f32 that is the same except next to a
// border between two results, where it is decided in 64 bits, so that the codes do not
// depend on how a quotient rounds.  A group with a NaN or an infinity stands for NaN.
#include <type_traits>

#include "../../include/starvector_sampling.h"
#include "sv_attention.h"
#include "sv_record.cuh"

namespace sv {
namespace {

constexpr int NT = 256;

struct WriteArgs {
  const void* in[2];
  int64_t i_row, i_head, i_tok;  // strides in elements
  unsigned char* cache[2];
  int64_t row, head, slot;  // strides in bytes
  const int32_t* lengths;
  int32_t* status;
  int32_t rows, kv_heads, dim, capacity, tokens;
};

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// x, which is off by up to three units in its last place, rounded to float16: false where those may decide (the 13
// bits that are dropped are near their middle), and for float16's subnormals.
__device__ __forceinline__ bool half_sure(float x, __half& h) {
  h = __float2half_rn(x);
  const uint32_t bits = __float_as_uint(x);
  return (bits & 0x1fffu) - (0x1000u - 8u) > 16u && (bits & 0x7fffffffu) >= 0x38800000u;
}

// (h - l) / 15 rounded once to float16.  Where the difference does not fit 64 bits its last bit stands for the rest: on
// neither side of a border of float16 (a fifteenth of which has 16 bits) does the quotient reach it then.
__device__ __noinline__ __half fifteenth(float h, float l) {
  double d = __dsub_rd((double)h, (double)l);
  if (d != __dsub_ru((double)h, (double)l)) d = __longlong_as_double(__double_as_longlong(d) | 1);
  return __double2half(d / 15.0);
}

__device__ __noinline__ bool above_exactly(float x, float mid, float scale, float half) {
  return (double)x > (double)mid + (double)half * (double)scale;  // exact: 11 bits and 16, 30 binades
}

// The whole number next to q = (x - mid) / scale, which was computed to within 2^-17: of the two next to it the upper
// one where x - mid is above (k + 1/2) scale, or equals it and the lower one is odd.  In f32 where that difference is exact
// (float16 and bfloat16 mostly; borders themselves are frequent there: one in 2000 values), otherwise in f64.
__device__ __forceinline__ float code_exactly(float x, float mid, float scale, float q) {
  const float k = floorf(q), half = k + 0.5f, t = x - mid, u = half * scale;
  const bool exact = fabsf(x) >= fabsf(mid) ? x - t == mid : t + mid == x;
  const bool odd = (int)k & 1;
  bool up = t > u || (t == u && odd);
  if (!exact) up = above_exactly(x, mid, scale, half) || (odd && !above_exactly(-x, -mid, -scale, half));
  return up ? k + 1.f : k;
}

// The smallest and the largest of eight values as they lie, NaN if one is.
__device__ __forceinline__ void extremes(const float4 (&v)[2], float& lo, float& hi) {
  lo = min_nan(min_nan(min_nan(v[0].x, v[0].y), min_nan(v[0].z, v[0].w)), min_nan(min_nan(v[1].x, v[1].y), min_nan(v[1].z, v[1].w)));
  hi = max_nan(max_nan(max_nan(v[0].x, v[0].y), max_nan(v[0].z, v[0].w)), max_nan(max_nan(v[1].x, v[1].y), max_nan(v[1].z, v[1].w)));
}
__device__ __forceinline__ void extremes(const uint4& v, float& lo, float& hi, __half) {
  auto f = [](uint32_t x) { return *reinterpret_cast<const __half2*>(&x); };
  const __half2 l = __hmin2_nan(__hmin2_nan(f(v.x), f(v.y)), __hmin2_nan(f(v.z), f(v.w)));
  const __half2 h = __hmax2_nan(__hmax2_nan(f(v.x), f(v.y)), __hmax2_nan(f(v.z), f(v.w)));
  lo = min_nan(__low2float(l), __high2float(l));
  hi = max_nan(__low2float(h), __high2float(h));
}
__device__ __forceinline__ void extremes(const uint4& v, float& lo, float& hi, __nv_bfloat16) {
  auto f = [](uint32_t x) { return *reinterpret_cast<const __nv_bfloat162*>(&x); };
  const __nv_bfloat162 l = __hmin2_nan(__hmin2_nan(f(v.x), f(v.y)), __hmin2_nan(f(v.z), f(v.w)));
  const __nv_bfloat162 h = __hmax2_nan(__hmax2_nan(f(v.x), f(v.y)), __hmax2_nan(f(v.z), f(v.w)));
  lo = min_nan(__low2float(l), __high2float(l));
  hi = max_nan(__low2float(h), __high2float(h));
}
__device__ __forceinline__ float2 two_of(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ float2 two_of(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// Eight values in a thread: as loaded, their extremes, as floats.
template <typename T> struct Eight {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void ends(float& lo, float& hi) const { extremes(v, lo, hi, T()); }
  __device__ __forceinline__ void floats(float (&f)[8]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 two = two_of(w[k], T());
      f[2 * k] = two.x;
      f[2 * k + 1] = two.y;
    }
  }
};
template <> struct Eight<float> {
  float4 v[2];
  __device__ __forceinline__ void load(const float* p) {
    v[0] = __ldg(reinterpret_cast<const float4*>(p));
    v[1] = __ldg(reinterpret_cast<const float4*>(p) + 1);
  }
  __device__ __forceinline__ void ends(float& lo, float& hi) const { extremes(v, lo, hi); }
  __device__ __forceinline__ void floats(float (&f)[8]) const {
    const float w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = w[k];
  }
};

// Where an item (one slot of one head, of keys or values) lies: blocks take slots of one
// unit (ONE: then everything but the slot is the same for the whole block), or units whole where these have few slots.
struct Item {
  int r, h, i;
  bool in;
};
template <bool ONE, int LPS_LOG2>
__device__ __forceinline__ Item item_at(int units_log2, int slots_log2, int kv_heads, int rows, int tokens) {
  // A block: 2^units_log2 units of 2^slots_log2 slots each.
  if (ONE) units_log2 = 0, slots_log2 = 8 - LPS_LOG2;
  const int item = threadIdx.x >> LPS_LOG2, unit = ((int)blockIdx.y << units_log2) + (ONE ? 0 : item >> slots_log2);
  Item x;
  x.r = unit / kv_heads;
  x.h = unit - x.r * kv_heads;
  x.i = ((int)blockIdx.x << slots_log2) + (item & ((1 << slots_log2) - 1));
  x.in = x.r < rows && x.i < tokens;
  return x;
}

template <typename T, int LPS_LOG2, bool ONE>  // 2^LPS_LOG2 threads per slot
__global__ void __launch_bounds__(NT) kv_quantize_kernel(const __grid_constant__ WriteArgs a, const int units_log2,
                                                         const int slots_log2) {
  wait_before();  // (launched while the kernel before it ends; the next one may be, too)
  launch_dependents();
  const int lane = threadIdx.x & ((1 << LPS_LOG2) - 1), y = lane & 1, i = lane >> 1;
  const Item it = item_at<ONE, LPS_LOG2>(units_log2, slots_log2, a.kv_heads, a.rows, a.tokens);
  int end = a.capacity, given = 0;
  if (it.in && a.lengths) {
    given = a.lengths[it.r];
    end = min(max(given, 0), a.capacity);
  }
  if (it.in && a.status && it.h == 0 && it.i == 0 && lane == 0 && blockIdx.z == 0)
    a.status[it.r] = a.lengths && given != end ? SV_ST_LENGTH : 0;
  const int blocks = (a.dim + 31) >> 5, slot = end - a.tokens + it.i;
  const bool in = it.in && slot >= 0 && i < blocks;  // (the shuffles need all lanes)
  const T* src = static_cast<const T*>(blockIdx.z ? a.in[1] : a.in[0]) + (it.r * a.i_row + it.h * a.i_head) + it.i * a.i_tok;
  Eight<T> x[2];
  bool has[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int d = 32 * i + 16 * e + 8 * y;
    has[e] = in && d < a.dim;
    if (has[e]) x[e].load(src + d);
  }
  float lo[2], hi[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    lo[e] = INFINITY;
    hi[e] = -INFINITY;
    if (has[e]) x[e].ends(lo[e], hi[e]);
  }
  constexpr bool wide = LPS_LOG2 == 3;  // groups of 32
  if (wide) {
    lo[0] = min_nan(lo[0], lo[1]);
    hi[0] = max_nan(hi[0], hi[1]);
  }
#pragma unroll
  for (int e = 0; e < (wide ? 1 : 2); ++e) {
    lo[e] = min_nan(lo[e], __shfl_xor_sync(0xffffffffu, lo[e], 1));
    hi[e] = max_nan(hi[e], __shfl_xor_sync(0xffffffffu, hi[e], 1));
  }
  uint32_t word[2] = {0u, 0u};
  uint32_t pair[2] = {0u, 0u};
  float scale = 0.f, mid = 0.f, inv = 0.f, base = 0.f;
  bool none = true, all_plain = true;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    if (!e || !wide) {
      // Without a value (dimensions past head_dim): zeros.  With one that is not finite: NaN.
      none = lo[e] > hi[e];
      const bool bad = !none && !(lo[e] > -INFINITY && hi[e] < INFINITY);
      const float l = fminf(fmaxf(lo[e], -kRecordMost), kRecordMost), h = fminf(fmaxf(hi[e], -kRecordMost), kRecordMost);
      __half s16, m16;
      if (!half_sure((h - l) * (1.f / 15.f), s16)) s16 = fifteenth(h, l);
      scale = __half2float(s16);
      if (!half_sure(fmaf(8.f, scale, l), m16)) m16 = __double2half((double)l + 8.0 * (double)scale);
      mid = __half2float(m16);
      inv = scale > 0.f ? __fdividef(1.f, scale) : 0.f;  // (to within two units in the last place)
      base = -mid * inv;
      // What is off from the whole number by rounding stays within 2^-17 in one step where mid is not many scales
      // away; and no code leaves its range where the extremes' do not.
      const bool plain = fabsf(base) <= 32.f && fmaf(hi[e], inv, base) < 7.4f && fmaf(lo[e], inv, base) > -8.4f;
      pair[e] = none ? 0u : bad ? 0x7e007e00u : (uint32_t)__half_as_ushort(s16) | (uint32_t)__half_as_ushort(m16) << 16;
      none = none || bad;
      all_plain = __all_sync(0xffffffffu, plain || none);
    }
    if (has[e] && !none) {
      // The whole number next to q by adding 1.5 2^23 (and 8): its last bits are the code then.
      constexpr float kAdd = 12582912.f + 8.f;
      constexpr uint32_t kBits = 0x4b400000u;
      float v[8], q[8], r[8], edge = 0.f;
      x[e].floats(v);
      if (!all_plain) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          v[k] = fminf(fmaxf(v[k], -kRecordMost), kRecordMost);
          q[k] = fminf(fmaxf((v[k] - mid) * inv, -8.f), 7.f);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) q[k] = fmaf(v[k], inv, base);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        r[k] = q[k] + kAdd;
        edge = fmaxf(edge, fabsf(q[k] - (r[k] - kAdd)));
      }
      if (edge > 0.5f - 0x1p-16f) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (fabsf(q[k] - (r[k] - kAdd)) > 0.5f - 0x1p-16f) r[k] = code_exactly(v[k], mid, scale, q[k]) + kAdd;
      }
      // Dimension 4 t + 2 a + b, t = 2 y + (k >> 2); the numbers' other bits are taken off the sum.
#pragma unroll
      for (int k = 0; k < 8; ++k) word[k >> 2] += __float_as_uint(r[k]) << 4 * (4 * (k & 1) + 2 * e + (k >> 1 & 1));
      word[0] -= kBits * (0x00110011u << 8 * e);
      word[1] -= kBits * (0x00110011u << 8 * e);
    }
  }
  if (!in) return;
  unsigned char* rec = (blockIdx.z ? a.cache[1] : a.cache[0]) + (it.r * a.row + it.h * a.head) + (int64_t)slot * a.slot;
  uint32_t* codes = reinterpret_cast<uint32_t*>(rec);
  codes[2 * y * blocks + i] = word[0];
  codes[(2 * y + 1) * blocks + i] = word[1];
  uint32_t* pairs = codes + 4 * blocks;
  if (wide) {
    if (y == 0) pairs[i] = pair[0];
    if (i == 0 && y == 1 && blocks == 3) pairs[3] = 0u;
  } else {
    pairs[2 * i + y] = pair[y];
    if (blocks == 1) pairs[2 + y] = 0u;
  }
}

template <typename T> __device__ __forceinline__ void store8(T* p, const float (&x)[8]);
template <> __device__ __forceinline__ void store8<float>(float* p, const float (&x)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
template <> __device__ __forceinline__ void store8<__half>(__half* p, const float (&x)[8]) {
  __half2 h[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) h[k] = __floats2half2_rn(x[2 * k], x[2 * k + 1]);
  *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
}
template <> __device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* p, const float (&x)[8]) {
  __nv_bfloat162 h[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) h[k] = __floats2bfloat162_rn(x[2 * k], x[2 * k + 1]);
  *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
}

// A thread takes PER slots, 2^slots_log2 apart: their words are on their way together.
template <typename T, int LPS_LOG2, int PER>
__global__ void __launch_bounds__(NT) kv_dequantize_kernel(const __grid_constant__ ReadArgs a, const int units_log2,
                                                           const int slots_log2) {
  wait_before();  // (launched while the kernel before it ends; the next one may be, too)
  launch_dependents();
  const int lane = threadIdx.x & ((1 << LPS_LOG2) - 1), y = lane & 1, i = lane >> 1;
  Item it = item_at<(PER > 1), LPS_LOG2>(units_log2, slots_log2, a.kv_heads, a.rows, a.tokens);
  if (PER > 1) it.i += (int)blockIdx.x * (PER - 1) << slots_log2;
  const int blocks = (a.dim + 31) >> 5;
  if (it.r >= a.rows || it.i >= a.tokens || i >= blocks) return;
  int end = a.capacity, given = 0;
  if (a.lengths) {
    given = a.lengths[it.r];
    end = min(max(given, 0), a.capacity);
  }
  if (a.status && it.h == 0 && it.i == 0 && lane == 0 && blockIdx.z == 0)
    a.status[it.r] = a.lengths && given != end ? SV_ST_LENGTH : 0;
  const int shift = a.newest ? end - a.tokens : 0;
  int start = 0, low = 0;
  if (a.seen) {
    start = a.starts ? min(max(a.starts[it.r], 0), end) : 0;
    low = a.window ? max(start, end - a.seen - a.window + 1) : start;
  }
  constexpr bool wide = LPS_LOG2 == 3;
  const unsigned char* unit = (blockIdx.z ? a.cache[1] : a.cache[0]) + it.r * a.row + it.h * a.head;
  T* out = static_cast<T*>(blockIdx.z ? a.out[1] : a.out[0]) +
           (((int64_t)it.r * a.kv_heads + it.h) * a.tokens + it.i) * a.dim;
  uint32_t word[PER][2], pair[PER][wide ? 1 : 2];
  bool writes[PER];
#pragma unroll
  for (int x = 0; x < PER; ++x) {
    const int place = it.i + (x << slots_log2), slot = place + shift;
    const bool in = slot >= 0 && slot < end;
    writes[x] = place < a.tokens && (!a.seen || (in && slot >= start && (slot >= low || slot < start + a.sinks)));
    word[x][0] = word[x][1] = pair[x][0] = pair[x][wide ? 0 : 1] = 0u;
    if (writes[x] && in) {
      const uint32_t* codes = reinterpret_cast<const uint32_t*>(unit + (int64_t)slot * a.slot);
      word[x][0] = __ldg(codes + 2 * y * blocks + i);
      word[x][1] = __ldg(codes + (2 * y + 1) * blocks + i);
      pair[x][0] = __ldg(codes + 4 * blocks + (wide ? i : 2 * i));
      if (!wide) pair[x][wide ? 0 : 1] = __ldg(codes + 4 * blocks + 2 * i + 1);
    }
  }
#pragma unroll
  for (int x = 0; x < PER; ++x) {
    if (!writes[x]) continue;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int d = 32 * i + 16 * e + 8 * y;
      if (d >= a.dim) break;
      const float2 sm = __half22float2(*reinterpret_cast<const __half2*>(&pair[x][wide ? 0 : e]));
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        // The nibble as the last bits of 2^23 + c.
        const uint32_t c = word[x][k >> 2] >> 4 * (4 * (k & 1) + 2 * e + (k >> 1 & 1)) & 15u;
        v[k] = fmaf(sm.x, __uint_as_float(0x4b000000u | c) - 8388616.f, sm.y);
      }
      T* to = out + ((int64_t)x << slots_log2) * a.dim + d;
      store8(to, v);
      if constexpr (!std::is_same<T, float>::value) {
        if (a.low && blockIdx.z == 0) {
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] -= (float)from_float<T>(v[k]);
          store8(static_cast<T*>(a.low) + (to - static_cast<T*>(a.out[0])), v);
        }
      }
    }
  }
}

// The grid of a kernel whose blocks take 2^(8 - lps_log2) slots: of one unit, or of several whole ones.
dim3 grid_of(int lps_log2, int64_t units, int tokens, bool both, int& units_log2, int& slots_log2) {
  slots_log2 = 0;
  while ((1 << slots_log2) < tokens && slots_log2 < 8 - lps_log2) ++slots_log2;
  units_log2 = 8 - lps_log2 - slots_log2;
  return dim3((unsigned)((tokens + (1 << slots_log2) - 1) >> slots_log2), (unsigned)((units + (1 << units_log2) - 1) >> units_log2),
              both ? 2u : 1u);
}

template <typename T> cudaError_t write_records(const WriteArgs& a, cudaStream_t stream) {
  int u, s;
  const int64_t units = (int64_t)a.rows * a.kv_heads;
  auto go = [&](auto one, auto many, int lps_log2) {
    const dim3 grid = grid_of(lps_log2, units, a.tokens, a.in[1] != nullptr, u, s);
    return launch_after(true, u == 0 ? one : many, grid, NT, 0, stream, a, u, s);
  };
  if (a.dim > 64) return go(kv_quantize_kernel<T, 3, true>, kv_quantize_kernel<T, 3, false>, 3);
  return a.dim > 32 ? go(kv_quantize_kernel<T, 2, true>, kv_quantize_kernel<T, 2, false>, 2)
                    : go(kv_quantize_kernel<T, 1, true>, kv_quantize_kernel<T, 1, false>, 1);
}

template <typename T> cudaError_t read_records(const ReadArgs& a, cudaStream_t stream) {
  int u, s;
  const int64_t units = (int64_t)a.rows * a.kv_heads;
  auto go = [&](auto one, auto four, int lps_log2) {
    // Four slots a thread where that leaves two blocks per SM (4 x 4096 slots of four heads of 128 in bfloat16 8.2 us, 10.9
    // with one; of one head 2.1 with one, 2.75 with four; float32 gains nothing: 23.2 us for the former, 19.8 with one).
    dim3 grid = grid_of(lps_log2, units, a.tokens, a.out[1] != nullptr, u, s);
    if (u == 0 && (int64_t)grid.x * grid.y * grid.z >= 8 * 148) {
      grid.x = (grid.x + 3) / 4;
      return launch_after(true, four, grid, NT, 0, stream, a, u, s);
    }
    return launch_after(true, one, grid, NT, 0, stream, a, u, s);
  };
  if (a.dim > 64) return go(kv_dequantize_kernel<T, 3, 1>, kv_dequantize_kernel<T, 3, 4>, 3);
  return a.dim > 32 ? go(kv_dequantize_kernel<T, 2, 1>, kv_dequantize_kernel<T, 2, 4>, 2)
                    : go(kv_dequantize_kernel<T, 1, 1>, kv_dequantize_kernel<T, 1, 4>, 1);
}

// What both calls take of a cache.
int check_records(const void* k, const void* v, int32_t rows, int32_t kv_heads, int32_t dim, int32_t capacity,
                  int32_t tokens, int64_t row, int64_t head, int64_t slot) {
  if (!k) return SV_E_ARG;
  if (rows < 1 || kv_heads < 1 || capacity < 1 || tokens < 0 || capacity > 1 << 29 || tokens > 1 << 29) return SV_E_SHAPE;
  if (dim < 8 || dim > kAttnMaxDim || dim % 8 || (int64_t)rows * kv_heads > 65535) return SV_E_SHAPE;
  if (row < 0 || head < 0 || slot < 0 || (capacity > 1 && slot == 0)) return SV_E_SHAPE;
  if (row % 16 || head % 16 || slot % 16) return SV_E_ALIGN;
  if (reinterpret_cast<uintptr_t>(k) % 16 || reinterpret_cast<uintptr_t>(v) % 16) return SV_E_ALIGN;
  return SV_OK;
}

// The bytes from the first entry of a strided array to behind its last.
template <int D> int64_t span_of(int64_t entry, const int64_t (&sizes)[D], const int64_t (&strides)[D]) {
  for (int d = 0; d < D; ++d) entry += (sizes[d] - 1) * strides[d];
  return entry;
}

bool overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return a && b && x < y + (uintptr_t)b_bytes && y < x + (uintptr_t)a_bytes;
}

}  // namespace

cudaError_t launch_read_records(const ReadArgs& a, cudaStream_t stream) {
  if (a.dtype == SV_F32) return read_records<float>(a, stream);
  return a.dtype == SV_F16 ? read_records<__half>(a, stream) : read_records<__nv_bfloat16>(a, stream);
}

}  // namespace sv

using namespace sv;

// See include/starvector_sampling.h.
extern "C" {

int32_t sv_kv_record_bytes(int32_t head_dim) {
  return head_dim < 8 || head_dim > kAttnMaxDim || head_dim % 8 ? 0 : record_bytes(head_dim);
}

int sv_kv_quantize(const void* keys, const void* values, int32_t dtype, int32_t rows, int32_t kv_heads, int32_t tokens,
                   int32_t head_dim, int64_t stride_row, int64_t stride_head, int64_t stride_token, void* cache_keys,
                   void* cache_values, int32_t capacity, int64_t cache_stride_row, int64_t cache_stride_head,
                   int64_t cache_stride_slot, const int32_t* lengths, int32_t* out_status, void* stream) {
  if (dtype != SV_F32 && dtype != SV_F16 && dtype != SV_BF16) return SV_E_DTYPE;
  if (!keys || (values != nullptr) != (cache_values != nullptr) || cache_keys == cache_values) return SV_E_ARG;
  const int rc = check_records(cache_keys, cache_values, rows, kv_heads, head_dim, capacity, tokens, cache_stride_row,
                               cache_stride_head, cache_stride_slot);
  if (rc) return rc;
  const int64_t e = dtype == SV_F32 ? 4 : 2;
  for (int64_t s : {stride_row, stride_head, stride_token})
    if (s < 0 || s * e % 16) return SV_E_ALIGN;
  if (reinterpret_cast<uintptr_t>(keys) % 16 || reinterpret_cast<uintptr_t>(values) % 16) return SV_E_ALIGN;
  // Every slot's record is written by its own threads, the keys' and the values'.
  const int64_t record = record_bytes(head_dim);
  const intptr_t apart = reinterpret_cast<intptr_t>(cache_values) - reinterpret_cast<intptr_t>(cache_keys);
  if (!entries_apart<4>(record, {rows, kv_heads, capacity, cache_values ? 2 : 1},
                        {cache_stride_row, cache_stride_head, cache_stride_slot, apart < 0 ? -apart : apart}))
    return SV_E_SHAPE;
  if (tokens == 0) return SV_OK;
  const int64_t in = span_of<3>(head_dim * e, {rows, kv_heads, tokens}, {stride_row * e, stride_head * e, stride_token * e});
  const int64_t out = span_of<3>(record, {rows, kv_heads, capacity}, {cache_stride_row, cache_stride_head, cache_stride_slot});
  for (const void* x : {keys, values})
    if (overlap(x, in, cache_keys, out) || overlap(x, in, cache_values, out)) return SV_E_ARG;
  WriteArgs a = {{keys, values}, stride_row, stride_head, stride_token,
                 {static_cast<unsigned char*>(cache_keys), static_cast<unsigned char*>(cache_values)},
                 cache_stride_row, cache_stride_head, cache_stride_slot, lengths, out_status,
                 rows, kv_heads, head_dim, capacity, tokens};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t err = dtype == SV_F32   ? write_records<float>(a, s)
                          : dtype == SV_F16 ? write_records<__half>(a, s)
                                            : write_records<__nv_bfloat16>(a, s);
  return err == cudaSuccess ? SV_OK : SV_E_CUDA;
}

int sv_kv_dequantize(const void* cache_keys, const void* cache_values, int32_t rows, int32_t kv_heads, int32_t head_dim,
                     int32_t capacity, int64_t cache_stride_row, int64_t cache_stride_head, int64_t cache_stride_slot,
                     const int32_t* lengths, int32_t tokens, void* keys, void* values, int32_t dtype,
                     int32_t* out_status, void* stream) {
  if (dtype != SV_F32 && dtype != SV_F16 && dtype != SV_BF16) return SV_E_DTYPE;
  if (!keys || (values != nullptr) != (cache_values != nullptr) || keys == values) return SV_E_ARG;
  const int rc = check_records(cache_keys, cache_values, rows, kv_heads, head_dim, capacity, tokens, cache_stride_row,
                               cache_stride_head, cache_stride_slot);
  if (rc) return rc;
  if (reinterpret_cast<uintptr_t>(keys) % 16 || reinterpret_cast<uintptr_t>(values) % 16) return SV_E_ALIGN;
  const int64_t in = span_of<3>(record_bytes(head_dim), {rows, kv_heads, capacity},
                                {cache_stride_row, cache_stride_head, cache_stride_slot});
  const int64_t out = (int64_t)rows * kv_heads * (tokens ? tokens : capacity) * head_dim * (dtype == SV_F32 ? 4 : 2);
  for (const void* x : {cache_keys, cache_values})
    if (overlap(x, in, keys, out) || overlap(x, in, values, out)) return SV_E_ARG;
  if (overlap(keys, out, values, out)) return SV_E_ARG;
  ReadArgs a = {};
  a.cache[0] = static_cast<const unsigned char*>(cache_keys);
  a.cache[1] = static_cast<const unsigned char*>(cache_values);
  a.row = cache_stride_row;
  a.head = cache_stride_head;
  a.slot = cache_stride_slot;
  a.out[0] = keys;
  a.out[1] = values;
  a.lengths = lengths;
  a.status = out_status;
  a.dtype = dtype;
  a.rows = rows;
  a.kv_heads = kv_heads;
  a.dim = head_dim;
  a.capacity = capacity;
  a.tokens = tokens ? tokens : capacity;
  a.newest = tokens != 0;
  return launch_read_records(a, static_cast<cudaStream_t>(stream)) == cudaSuccess ? SV_OK : SV_E_CUDA;
}

}  // extern "C"
