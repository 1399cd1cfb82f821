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
// over the 16 lanes that hold a block
__device__ __forceinline__ float fp8_block_largest(float a) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) a = fp8_max(a, __shfl_xor_sync(0xffffffffu, a, o));
  return fp8_max(a, FP8_TINY);
}
__device__ __forceinline__ uint8_t fp8_one(float v) { return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); }
// eight numbers times `inv`, as eight bytes
__device__ __forceinline__ uint2 fp8_eight(const float (&v)[8], float inv) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i] * inv, v[2 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

}  // namespace
