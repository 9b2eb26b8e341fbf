// MXFP4 (OCP microscaling, E2M1 elements, one UE8M0 scale for each block of
// 32 along a row) as device functions: used by the quantisation kernel
// (mxfp4.cu) and by the projection over MXFP4 weights (linear_mxfp4.cu).
//
//   e = floor(log2(max |x|)) - 2 (2 = the exponent of E2M1's largest value),
//   clamped to [-127, 127];  scale code = e + 127;
//   element = E2M1 nearest to x 2^-e, ties to even, saturating at +-6.
// floor(log2) is the exponent field of the maximum's fp32 bits, so the scale
// costs no logarithm; 2^-e has the exponent field 254 - code and the product
// with it is exact, so the one rounding is the E2M1 conversion itself.  A
// maximum below 2^-124 (zero included) takes code 0.  A block with a NaN or
// an infinity takes code 255, UE8M0's NaN, and zero elements: whatever is
// made of the block is NaN.
#pragma once

#include "common.cuh"
#include <cuda_fp16.h>
#include <cuda_fp4.h>

namespace dsa {
namespace mx {

constexpr int kBlock = 32;
constexpr int kVec = 8;  // elements a lane holds; a block is 4 neighbouring lanes

// 8 consecutive elements as fp32
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float* v) {
  bf16x8_to_f32(__ldg(reinterpret_cast<const uint4*>(p)), v);
}
__device__ __forceinline__ void load8(const __half* p, float* v) {
  const uint4 w = __ldg(reinterpret_cast<const uint4*>(p));
  const __half2* h = reinterpret_cast<const __half2*>(&w);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void load8(const float* p, float* v) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

// The scale code of the block whose 32 elements this lane and its three
// neighbours hold (every lane of the warp calls it).  The fp32 bits without
// the sign order as integers, NaN and infinity above every number.
__device__ __forceinline__ uint32_t scale_code(const float* v) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < kVec; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  const int field = int(m >> 23);
  return field == 255 ? 255u : uint32_t(max(field - 2, 0));
}

// this lane's 8 elements as E2M1, two a byte, the even element in the low half
__device__ __forceinline__ uint32_t codes8(const float* v, uint32_t sc) {
  if (sc == 255u) return 0u;
  const float inv = __uint_as_float((254u - sc) << 23);
  uint32_t c = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_fp4x2_storage_t b =
        __nv_cvt_float2_to_fp4x2(make_float2(v[2 * i] * inv, v[2 * i + 1] * inv), __NV_E2M1, cudaRoundNearest);
    c |= uint32_t(b) << (8 * i);
  }
  return c;
}

// the values the codes stand for
__device__ __forceinline__ void values8(uint32_t codes, uint32_t sc, float* v) {
  const float s = sc == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float(sc ? sc << 23 : 0x00400000u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2(__nv_fp4x2_storage_t((codes >> (8 * i)) & 0xffu), __NV_E2M1);
    const float2 f = __half22float2(__half2(h));
    v[2 * i] = f.x * s;
    v[2 * i + 1] = f.y * s;
  }
}

}  // namespace mx
}  // namespace dsa
