// What the tensor-core attention kernels share: operand packing, masks as bit
// words, tensor maps.
#pragma once

#include "window_attn.cuh"

#include "launch.cuh"
#include "tma.cuh"
#include "tmap.cuh"
#include "umma.cuh"

namespace mr {

constexpr int kTileBytes = 16384;  // [128 rows][64 2-byte elements], 128-byte swizzle
template <typename T> struct Fmt;
template <> struct Fmt<__nv_bfloat16> {
  static constexpr int id = 1;
  static __device__ uint32_t pack(float a, float b) {
    __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&r);
  }
  static __device__ float2 unpack(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v)); }
};
template <> struct Fmt<__half> {
  static constexpr int id = 0;
  static __device__ uint32_t pack(float a, float b) {
    __half2 r = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&r);
  }
  static __device__ float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
};

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// bits [a, b) of a 32-bit word, whatever the bounds
__device__ __forceinline__ uint32_t bits(int a, int b) {
  const uint32_t hi = b >= 32 ? 0xffffffffu : b <= 0 ? 0u : (1u << b) - 1;
  const uint32_t lo = a >= 32 ? 0xffffffffu : a <= 0 ? 0u : (1u << a) - 1;
  return hi & ~lo;
}

// rows of one head of [T, H, Dh] as (Dh, H, T); columns at and behind Dh and rows behind T read as zero
static inline int head_map(CUtensorMap* m, const void* p, CUtensorMapDataType dt, const AttnArgs& A, int H, int64_t ts,
                           int64_t hs, int rows) {
  return make_tmap_3d(m, p, dt, 2, A.Dh, H, A.T, hs * 2, ts * 2, 64, 1, rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace mr
