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

// 8 e4m3 codes times their scale, rounded to bf16 once.  e4m3 -> fp16 is
// exact, fp16 -> fp32 too, and the fp32 product is the one kv_window_write
// rounds.  (A code is never NaN: kv_quant_write marks a block that holds a
// NaN or an infinity by a NaN scale.)
__device__ __forceinline__ void values8(uint2 codes, float s, float* v) {
  const uint32_t w[2] = {codes.x, codes.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t((w[i >> 1] >> (16 * (i & 1))) & 0xffffu), __NV_E4M3);
    const float2 f = __half22float2(__half2(h));
    v[2 * i] = f.x * s;
    v[2 * i + 1] = f.y * s;
  }
}

__device__ __forceinline__ uint4 bf16_values8(uint2 codes, float s) {
  float v[8];
  values8(codes, s, v);
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

}  // namespace kvq
}  // namespace dsa
