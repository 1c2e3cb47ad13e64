// The 8-bit paged KV cache: codes, scales and layout, shared by the kernels that write it
// (qk_norm_rope.cu) and read it (attention_q8.cu).
//
// Codes are int8 (-127..127) or float8 e4m3, one float32 scale per (layer, block, kv head):
// a stored value is code * scale.  A cache is [layers, num_blocks, nkv, 16, head_dim], so the
// 16 tokens of one block and head are one run of 16 * head_dim bytes (2 KB at 128), which a
// reader fetches with full 128-byte lines; the scales are [layers, num_blocks, nkv].
//
// The scale of a tile is amax / 127 or amax / 448 over the values it was written from.  A
// scale of 0 stands for a tile of zeros (amax below 2^-126 times the largest code), NaN for
// one that a value which is not finite was written to.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace b2 {

constexpr int kQ8Block = 16;  // tokens per block
constexpr float kQ8Tiny = 1.17549435e-38f;  // 2^-126: below it 1 / scale is not finite

inline bool valid_q8_dtype(int d) { return d == B2_I8 || d == B2_E4M3; }

template <int CODE>
struct Q8;

template <>
struct Q8<B2_I8> {
  static constexpr float kTop = 127.f;
  // Four codes in the bytes of w, lowest first.
  static __device__ __forceinline__ void decode4(uint32_t w, float (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (float)(int8_t)(w >> (8 * i));
  }
  static __device__ __forceinline__ uint32_t encode4(const float (&v)[4]) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = max(-127, min(127, __float2int_rn(v[i])));
      w |= (uint32_t)(c & 0xff) << (8 * i);
    }
    return w;
  }
};

template <>
struct Q8<B2_E4M3> {
  static constexpr float kTop = 448.f;
  static __device__ __forceinline__ void decode4(uint32_t w, float (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * i)), __NV_E4M3);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ uint32_t encode4(const float (&v)[4]) {  // to nearest, saturating
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[0], v[1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[2], v[3]), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  }
};

// Element offset of the tile (block, head) of one layer's cache, and of its scale.
__device__ __forceinline__ int64_t q8_tile(int64_t block, int nkv, int head, int hd) {
  return (block * nkv + head) * (int64_t)(kQ8Block * hd);
}
__device__ __forceinline__ int64_t q8_scale(int64_t block, int nkv, int head) { return block * nkv + head; }

// x, or the largest number where x is infinite; a NaN stays one.
__device__ __forceinline__ float q8_finite(float x) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(3.402823466e38f));
  return y;
}

}  // namespace b2
