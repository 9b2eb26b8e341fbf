// The FP8 latent cache: one record a row (a token's latent vector of D dims,
// the last rope_dim of them rotary),
//   [D - rope_dim e4m3 codes][rope_dim bf16][(D - rope_dim) / 64 fp32 scales][zeros to a multiple of 32 B]
// 448 + 128 + 28 -> 608 B for D = 512, rope_dim = 64, against 1024 B of bf16.
// Whole 32-byte sectors, so writing a record reads nothing back and a
// gathered record touches no other row's sectors.  The value of a code is
// bf16(float(code) * scale): what dsa_kv_window_write stores for the same row.
#pragma once

#include "common.cuh"
#include <cuda_fp16.h>

namespace dsa {
namespace kvq {

constexpr int kBlock = 64;  // dims a scale covers

__host__ __device__ constexpr int row_bytes(int nope, int rope) {
  return (nope + 2 * rope + 4 * (nope / kBlock) + 31) / 32 * 32;
}

// 8 e4m3 codes times their scale in fp32: e4m3 -> fp16 -> fp32 is exact, so
// the product is the one kv_window_write rounds.  (A code is never NaN:
// kv_quant_write marks a block that holds a NaN or an infinity by a NaN
// scale.)  Two products an instruction (mul.f32x2).
__device__ __forceinline__ void values8(uint2 codes, float s, float* v) {
  const uint32_t w[2] = {codes.x, codes.y};
  uint64_t s2;
  asm("mov.b64 %0, {%1, %1};" : "=l"(s2) : "f"(s));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t h[2];
    asm("{\n\t.reg .b16 lo, hi;\n\t"
        "mov.b32 {lo, hi}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, lo;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
        : "=r"(h[0]), "=r"(h[1])
        : "r"(w[i]));
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
      uint64_t x;
      asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(f.x), "f"(f.y));
      asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(x) : "l"(x), "l"(s2));
      asm("mov.b64 {%0, %1}, %2;" : "=f"(v[4 * i + 2 * j]), "=f"(v[4 * i + 2 * j + 1]) : "l"(x));
    }
  }
}

__device__ __forceinline__ uint4 bf16_values8(uint2 codes, float s) {
  float v[8];
  values8(codes, s, v);
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

}  // namespace kvq
}  // namespace dsa
