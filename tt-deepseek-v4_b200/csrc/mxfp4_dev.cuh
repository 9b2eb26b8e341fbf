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
constexpr int kVec = 8;  // a lane's elements come in eights

// A lane's 8 consecutive elements as they lie in memory.
template <typename T>
struct Vec8 {
  uint4 w[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Vec8<T> load8(const T* p) {
  Vec8<T> r;
#pragma unroll
  for (int i = 0; i < int(sizeof(T) / 2); ++i) r.w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  return r;
}
template <typename T>
__device__ __forceinline__ Vec8<T> zero8() {
  Vec8<T> r;
#pragma unroll
  for (int i = 0; i < int(sizeof(T) / 2); ++i) r.w[i] = make_uint4(0, 0, 0, 0);
  return r;
}

__device__ __forceinline__ __nv_bfloat162 as_bf162(uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); }
__device__ __forceinline__ uint32_t as_u32(__nv_bfloat162 h) { return *reinterpret_cast<const uint32_t*>(&h); }

// eight fp32 values as E2M1, two a byte, the first in the low half
__device__ __forceinline__ uint32_t e2m1x8(const float* f) {
  uint32_t c;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(c)
      : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
  return c;
}

// A block on 4 / H neighbouring lanes, H eights each: its scale code (every
// lane of the warp calls it) and the E2M1 codes of this lane's eights.  With
// one eight a lane the shuffles and the scale's arithmetic bound 16-bit
// inputs, not the bytes (4096 x 8192 bf16 into the projection's tiles: 17.4
// us; loads and stores alone 12.3).
// fp32 and fp16: the fp32 bits without the sign order as integers, NaN and
// infinity above every number.
template <typename T, int H>
__device__ __forceinline__ void quant(const Vec8<T> (&x)[H], uint32_t& sc, uint32_t (&codes)[H]) {
  float v[H][kVec];
  uint32_t m = 0;
#pragma unroll
  for (int h = 0; h < H; ++h) {
    if constexpr (sizeof(T) == 4) {
      const uint32_t w[8] = {x[h].w[0].x, x[h].w[0].y, x[h].w[0].z, x[h].w[0].w,
                             x[h].w[1].x, x[h].w[1].y, x[h].w[1].z, x[h].w[1].w};
#pragma unroll
      for (int i = 0; i < kVec; ++i) v[h][i] = __uint_as_float(w[i]);
    } else {
      const __half2* p = reinterpret_cast<const __half2*>(&x[h].w[0]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(p[i]);
        v[h][2 * i] = f.x;
        v[h][2 * i + 1] = f.y;
      }
    }
#pragma unroll
    for (int i = 0; i < kVec; ++i) m = max(m, __float_as_uint(v[h][i]) & 0x7fffffffu);
  }
#pragma unroll
  for (int o = 1; o < 4 / H; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  const int field = int(m >> 23);
  sc = field == 255 ? 255u : uint32_t(max(field - 2, 0));
  const float inv = __uint_as_float((254u - sc) << 23);
#pragma unroll
  for (int h = 0; h < H; ++h) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[h][i] *= inv;
    codes[h] = sc == 255u ? 0u : e2m1x8(v[h]);
  }
}
// bf16: maximum and scaling two elements an instruction (a power of two, so
// exact where the code is not zero)
template <int H>
__device__ __forceinline__ void quant(const Vec8<__nv_bfloat16> (&x)[H], uint32_t& sc, uint32_t (&codes)[H]) {
  __nv_bfloat162 m = as_bf162(0u);
#pragma unroll
  for (int h = 0; h < H; ++h) {
    const uint32_t w[4] = {x[h].w[0].x, x[h].w[0].y, x[h].w[0].z, x[h].w[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __hmax2_nan(m, __habs2(as_bf162(w[i])));
  }
#pragma unroll
  for (int o = 1; o < 4 / H; o <<= 1) m = __hmax2_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  const uint32_t mb = as_u32(m);
  // the exponent field orders as the number does, NaN and infinity 255
  const int field = int(max((mb >> 7) & 0xffu, (mb >> 23) & 0xffu));
  sc = field == 255 ? 255u : uint32_t(max(field - 2, 0));
  const __nv_bfloat162 inv = as_bf162(((254u - sc) << 7) * 0x10001u);
#pragma unroll
  for (int h = 0; h < H; ++h) {
    const uint32_t w[4] = {x[h].w[0].x, x[h].w[0].y, x[h].w[0].z, x[h].w[0].w};
    float f[kVec];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t y = as_u32(__hmul2(as_bf162(w[i]), inv));
      f[2 * i] = __uint_as_float(y << 16);
      f[2 * i + 1] = __uint_as_float(y & 0xffff0000u);
    }
    codes[h] = sc == 255u ? 0u : e2m1x8(f);
  }
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
