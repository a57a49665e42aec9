// sv_record.cuh -- the cache held in 4 bits: one record per slot of one key/value head.
//
// P = head_dim rounded up to 32.  A record is P / 2 bytes of codes, then four pairs of
// float16 (scale, mid) of groups of dimensions: 32 of them where P >= 96, 16 below; pairs
// without a group are zero.  A dimension's value is mid + scale (c - 8), c its code.
// 32-bit word t P / 32 + i of the codes (t < 4) holds eight of block i's 32 dimensions:
// nibble 4 b + 2 e + a that of dimension 32 i + 16 e + 4 t + 2 a + b, zero past head_dim.
// So thread t of a quarter warp finds its operands of a product over 16 dimensions (two
// pairs of neighbours) with two masks, in one vector of the record; records are
// multiples of 16 bytes, so that what moves slots moves them as they are.
#pragma once
#include <cstdint>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace sv {

__host__ __device__ constexpr int record_dims(int dim) { return (dim + 31) / 32 * 32; }
__host__ __device__ constexpr int record_codes(int dim) { return record_dims(dim) / 2; }
__host__ __device__ constexpr int record_bytes(int dim) { return record_codes(dim) + 16; }

constexpr float kRecordMost = 32768.f;  // finite values beyond count as this: what they stand for stays in float16

// Slots of records read into plain values.
struct ReadArgs {
  const unsigned char* cache[2];  // keys, values (may be null)
  int64_t row, head, slot;        // strides in bytes
  void* out[2];                   // [rows][kv_heads][tokens][dim]
  void* low;                      // with 16-bit types: what the keys' rounding left, rounded; or null
  const int32_t *lengths, *starts;
  int32_t* status;
  int32_t dtype, rows, kv_heads, dim, capacity;
  int32_t tokens;   // places of out; place i holds slot
  int32_t newest;   // ... length - tokens + i if newest, i if not
  // Places without a slot of the row become zeros.  seen > 0 (with newest = 0): only the slots
  // that one of the row's last `seen` queries sees under the window are written at all.
  int32_t seen, window, sinks;
};
cudaError_t launch_read_records(const ReadArgs& a, cudaStream_t stream);

}  // namespace sv
