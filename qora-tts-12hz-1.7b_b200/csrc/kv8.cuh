// kv8.cuh -- device helpers of the 8-bit paged cache kernels.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"
#include "kv8.h"

namespace qtts {
namespace {

constexpr unsigned kFull = 0xffffffffu;

// ---- four consecutive elements of a row --------------------------------------
__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 load4(const __half* p) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                     __uint_as_float(u.y & 0xffff0000u));
}
__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void store4(__half* p, float4 v) {
  *reinterpret_cast<uint2*>(p) =
      make_uint2(half2_bits(__floats2half2_rn(v.x, v.y)), half2_bits(__floats2half2_rn(v.z, v.w)));
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, float4 v) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
  *reinterpret_cast<uint2*>(p) =
      make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

__device__ __forceinline__ void raise(int* flags, int bit) {
  if (flags) atomicOr(flags, bit);
}

// codes and scale of (page, K = 0 / V = 1, kv head)
__device__ __forceinline__ int8_t* block_codes(const qtts_kv8_cache& c, int page, int which, int h) {
  return c.codes + (size_t)page * c.page_stride + (size_t)(which * c.kv_heads + h) * kKv8Page * c.head_dim;
}
__device__ __forceinline__ float* block_scale(const qtts_kv8_cache& c, int page, int which, int h) {
  return c.scales + (size_t)page * c.scale_stride + which * c.kv_heads + h;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two bytes of w ^ 0x80808080 (a code + 128) become the f16 pair 1024 + (code +
// 128) by a byte permute onto 0x64; subtracting 1152 is exact.
__device__ __forceinline__ uint32_t half2_of(uint32_t biased, uint32_t sel) {
  uint32_t r = __byte_perm(biased, 0x64646464u, sel);
  const __half2 h = __hsub2(*reinterpret_cast<__half2*>(&r), __half2half2(__ushort_as_half(0x6480)));
  return half2_bits(h);
}
// Four codes of a word (little end first) as two f16 pairs.
__device__ __forceinline__ uint2 halves_of(uint32_t codes) {
  const uint32_t u = codes ^ 0x80808080u;
  return make_uint2(half2_of(u, 0x4140), half2_of(u, 0x4342));
}
// scale = fr * 2^ev with fr in [1, 2) (0, subnormal, infinite and NaN scales keep fr = what is left)
__device__ __forceinline__ void split_scale(float scale, float& ev, float& fr) {
  const int b = __float_as_int(scale), x = (b >> 23) & 255;
  ev = x == 0 ? -126.0f : x == 255 ? 0.0f : (float)(x - 127);
  fr = x == 0 ? scale * 0x1p126f : x == 255 ? scale : __int_as_float((b & 0x807fffff) | 0x3f800000);
}

}  // namespace
}  // namespace qtts
