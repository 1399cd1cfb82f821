// Numbers in e4m3 with a float32 scale for every 128 of a row: what the kernels that write and read them share.
//
// A block of 128 columns (the last of a row may be shorter) is held as q = e4m3(v * (448 / a)) and the scale a / 448, a the block's
// largest |v| but at least 2^-100, so that a block of zeros (or of numbers that vanish beside any other block) has finite scales both ways.
// The largest number falls on 448, the largest e4m3; rounding is to nearest even, off by at most 2^-4 of a number of normal size.  A NaN
// or an infinity makes the block's scale one too, so it stays visible in all that is computed from the block.
// Scales lie [blocks][rows]: the scales of one block for neighbouring rows, which a product reads together, are neighbours.
#pragma once
#include <cuda_fp8.h>
#include "common.cuh"

namespace {

constexpr int FP8_BLOCK = 128;
constexpr float FP8_TOP = 448.f;
constexpr float FP8_TINY = 7.888609052210118e-31f;      // 2^-100

// the larger of the two, NaN if one of them is
__device__ __forceinline__ float fp8_max(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float fp8_largest(const float (&v)[8]) {
  float a = fabsf(v[0]);
#pragma unroll
  for (int e = 1; e < 8; ++e) a = fp8_max(a, fabsf(v[e]));
  return a;
}
// two numbers at a time
__device__ __forceinline__ float2 fp8_add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fp8_mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fp8_fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
// over the 16 lanes that hold a block
__device__ __forceinline__ float fp8_block_largest(float a) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) a = fp8_max(a, __shfl_xor_sync(0xffffffffu, a, o));
  return fp8_max(a, FP8_TINY);
}
// 448 / a and a / 448 to an ulp or two.  (The reciprocal of a / 256, so that those of the largest numbers are no denormals, which it makes zero.)
__device__ __forceinline__ float fp8_up(float a) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a * 0.00390625f));
  return r * (FP8_TOP * 0.00390625f);
}
__device__ __forceinline__ float fp8_scale(float a) { return a * (1.f / FP8_TOP); }
__device__ __forceinline__ uint8_t fp8_one(float v) { return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); }
// eight numbers times `inv`, as eight bytes
__device__ __forceinline__ uint2 fp8_eight(const float (&v)[8], float inv) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = __nv_cvt_float2_to_fp8x2(fp8_mul2(make_float2(v[2 * i], v[2 * i + 1]), make_float2(inv, inv)), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

}  // namespace
