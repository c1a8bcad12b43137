// sa_kv4.cuh -- the 4-bit cache entry shared by the pack, unpack and
// attention kernels.
//
// An entry is one (block of 32 tokens, KV head): 36 * D bytes,
//
//   [16 D  key codes][16 D  value codes][2 D  key scales][2 D  value scales].
//
// A row is quantised in groups of 64 elements, each with an FP16 step and an
// FP16 minimum: value = step * code + minimum, code in 0..15. The orders below
// are those in which a warp's m16n8k16 matrix fragments want the data, so that
// the attention reads every code with a 16-byte load per lane and splits words
// into operand registers with one AND each:
//
//  * keys (matrix rows = tokens): row r is D / 2 contiguous bytes. Fragment
//    column owner t (0..3) holds elements 16t .. 16t+15 of every group, the
//    groups side by side: 8 bytes a group, 8 * (D / 64) bytes a t.
//  * values (matrix columns = tokens): tokens 2i and 2i+1 share a pair row of
//    D bytes, since a register holds two consecutive tokens of one element.
//    Fragment row owner g (0..7) holds elements 8g .. 8g+7 of every group;
//    a 32-bit word is 4 elements of the even token, then of the odd one.
//  * key scales (step, minimum): [group][r % 8][r / 8], so that the rows of
//    one lane (r, r + 8, r + 16, r + 24) are 16 contiguous bytes.
//  * value scales: all steps [group][32], then all minima [group][32], tokens
//    in the order (t, j, h, b) of r = 16j + 8h + 2t + b: the eight tokens of
//    a column owner t are 16 contiguous bytes.
#pragma once

#include <cuda_bf16.h>

#include "sa_device.cuh"

namespace sa {

constexpr int kKv4Group = 64;  // elements that share a step and a minimum

__host__ __device__ constexpr int kv4_entry_bytes(int d) { return 36 * d; }
__host__ __device__ constexpr int kv4_value_codes(int d) { return 16 * d; }
__host__ __device__ constexpr int kv4_key_scales(int d) { return 32 * d; }
__host__ __device__ constexpr int kv4_value_scales(int d) { return 34 * d; }

// Byte of the 8 key bytes of elements [64 * group + 16t, + 16) of row r.
__device__ __forceinline__ int kv4_key_at(int d, int r, int group, int t) {
  return r * (d >> 1) + 8 * (d / kKv4Group) * t + 8 * group;
}
// Byte of the 16-bit piece with elements [64 * group + 8g + 4w + 2h, + 2) of row r.
__device__ __forceinline__ int kv4_value_at(int d, int r, int group, int g, int w, int h) {
  return kv4_value_codes(d) + (r >> 1) * d + 8 * (d / kKv4Group) * g + 8 * group + 4 * w +
         2 * (r & 1) + h;
}
// Byte of the (step, minimum) pair of a key group.
__device__ __forceinline__ int kv4_key_scale_at(int d, int r, int group) {
  return kv4_key_scales(d) + 4 * ((group * 8 + (r & 7)) * 4 + (r >> 3));
}
// Byte of a value group's step; its minimum is d bytes further on.
__device__ __forceinline__ int kv4_value_scale_at(int d, int r, int group) {
  const int order = ((r & 7) >> 1) * 8 + (r >> 4) * 4 + ((r >> 3) & 1) * 2 + (r & 1);
  return kv4_value_scales(d) + 64 * group + 2 * order;
}

// Minimum and maximum that are NaN if an operand is.
__device__ __forceinline__ float min_nan(float a, float b) {
  float c;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
  return c;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float c;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
  return c;
}

// The largest FP16 number, where FP16 outputs stop (NaN stays). The step is rounded up, so
// the code 15 of a row next to the range's end stands for up to 65,616, which would be
// infinite in FP16. Held values are not below the minimum, so not below -65,504.
constexpr float kHalfMost = 65504.0f;

// ---- element types of the calls (SA_TYPE_*) -------------------------------------

template <int TYPE>
struct Kv4Type;
template <>
struct Kv4Type<SA_TYPE_F32> {
  using T = float;
  static __device__ __forceinline__ float load(T x) { return x; }
  static __device__ __forceinline__ T store(float x) { return x; }
};
template <>
struct Kv4Type<SA_TYPE_F16> {
  using T = __half;
  static __device__ __forceinline__ float load(T x) { return __half2float(x); }
  static __device__ __forceinline__ T store(float x) { return __float2half_rn(x); }
};
template <>
struct Kv4Type<SA_TYPE_BF16> {
  using T = __nv_bfloat16;
  static __device__ __forceinline__ float load(T x) { return __bfloat162float(x); }
  static __device__ __forceinline__ T store(float x) { return __float2bfloat16_rn(x); }
};

}  // namespace sa
