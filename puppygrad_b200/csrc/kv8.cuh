// What the kernels over the 8-bit cache share: rows of a sequence, pages, conversions.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "device_util.cuh"
#include "serving.h"

namespace pg {
namespace {

// Rows [first, first + n) of sequence b. Whatever row_start holds, they lie within the call's rows.
struct SeqRows {
  int first, n;
};
__device__ __forceinline__ SeqRows seq_rows(const int* row_start, int rows, int b) {
  if (!row_start) return {b, 1};
  const int r0 = min(max(row_start[b], 0), rows), r1 = min(max(row_start[b + 1], r0), rows);
  return {r0, r1 - r0};
}

// Page of logical page `lp` of sequence b, -1 where there is none.
__device__ __forceinline__ int page_of(const Kv8View& c, int b, int lp) {
  if (lp < 0 || lp >= c.pages_per_seq) return -1;
  const int page = c.table[(size_t)b * c.pages_per_seq + lp];
  return (unsigned)page < (unsigned)c.n_pages ? page : -1;
}

// Softmax weights go to FP16 as up to 2^15, its upper end: their rounding, 2^-25 below its normal numbers, is then 2^-40 of the largest, and a long tail
// of small weights is not lost. Maxima are rounded up and what is taken from an exponent down, so that no weight is larger.
constexpr float WEIGHT_BITS = 15.f;

// Two e4m3 codes (low and high byte) as FP16, exact.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
  uint32_t r;
  asm("{\n.reg .b16 t;\ncvt.u16.u32 t, %1;\ncvt.rn.f16x2.e4m3x2 %0, t;\n}" : "=r"(r) : "r"(two));
  return r;
}
// Rounded to nearest even, kept within +-448; `a` in the low byte.
__device__ __forceinline__ uint32_t f32x2_to_e4m3x2(float a, float b) {
  uint32_t r;
  asm("{\n.reg .b16 t;\ncvt.rn.satfinite.e4m3x2.f32 t, %2, %1;\ncvt.u32.u16 %0, t;\n}" : "=r"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t f32x4_to_e4m3x4(float a, float b, float c, float d) {
  return f32x2_to_e4m3x2(a, b) | f32x2_to_e4m3x2(c, d) << 16;
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_f16(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }

}  // namespace
}  // namespace pg
