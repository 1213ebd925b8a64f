// The paged 8-bit cache: e4m3 codes, one scale a page and head, and how packed rows find their request.
#pragma once

#include "elem.cuh"

namespace dspark {
namespace paged {

// Device status of what an append dropped (no room, or a page id outside the pool) and of pages outside the
// pool that an attention did not see; shared memory that begins off a 1024-byte boundary.
constexpr int kErrAppendPage = 0x206, kErrAttnPage = 0x207, kErrAlign = 0x208;

// Two codes (the low byte first) as two fp16 values: every e4m3 value is an fp16 one.
__device__ __forceinline__ uint32_t e4m3_to_f16(uint32_t codes) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}
__device__ __forceinline__ uint32_t e4m3_to_f16_hi(uint32_t codes) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}

// Four values as codes, round to nearest even, at most 448; NaN stays NaN.
__device__ __forceinline__ uint32_t f32_to_e4m3(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tcvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\t"
      "mov.b32 %0, {l, h};\n\t}"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}

// The exponent of the smallest power of two s with amax <= 448 s = 1.75 * 2^8 s, from -64 to 64.
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = int(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u);
  return min(max(e, -64), 64);
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// Packed rows of request b, held to the R that there are.
__device__ __forceinline__ int first_row(const int32_t* cu_rows, int b, int R) { return min(max(cu_rows[b], 0), R); }

// Of n values that rise with their index, f(0) <= x: the last index with f(i) <= x. A warp together.
template <typename F>
__device__ __forceinline__ int last_at_most(int n, int x, F f) {
  const int lane = threadIdx.x & 31;
  int lo = 0;
  while (n > 1) {
    const int step = (n + 31) >> 5, i = lane * step;
    const unsigned hit = __ballot_sync(0xffffffffu, i < n && f(lo + i) <= x);
    const int k = max(31 - __clz(hit), 0);  // (no hit: f does not rise; the first then)
    lo += k * step;
    n = min(step, n - k * step);
  }
  return lo;
}

}  // namespace paged
}  // namespace dspark
