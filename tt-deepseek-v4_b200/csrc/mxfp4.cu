// MXFP4 quantisation of a matrix along its rows (formulas in mxfp4_dev.cuh).
//
// A lane holds 8 consecutive elements, 4 lanes a block of 32, so the block's
// maximum is two shuffles and nothing touches shared memory.  The kernel is
// an HBM stream (2 or 4 B in; 0.5 B of codes, 1/32 B of scales and, on
// request, the 2 or 4 B of the values the codes stand for out).
#include "mxfp4_dev.cuh"

namespace dsa {
namespace mx {

__device__ __forceinline__ void store8(__nv_bfloat16* p, const float* v) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ void store8(__half* p, const float* v) {
  __half2 h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
}
__device__ __forceinline__ void store8(float* p, const float* v) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

constexpr int kThreads = 256;
constexpr int kUnroll = 2;  // 8-element chunks a thread has in flight

// Chunks [0, total) of 8 elements in row order, total a multiple of 4; the
// codes and scales are contiguous, x and out have row strides.
template <typename T>
__global__ void __launch_bounds__(kThreads) mxfp4_quant_kernel(const T* __restrict__ x, int64_t ld_x,
                                                               T* __restrict__ out, int64_t ld_out,
                                                               uint32_t* __restrict__ codes,
                                                               uint8_t* __restrict__ scales, int64_t total,
                                                               int row_chunks) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t step = int64_t(gridDim.x) * kThreads * kUnroll;
  const bool flat = ld_x == int64_t(row_chunks) * kVec && (!out || ld_out == ld_x);
  // whole warps stay in the loop: the block maximum is a warp shuffle
  for (int64_t c0 = int64_t(blockIdx.x) * kThreads * kUnroll; c0 < total; c0 += step) {
    Vec8<T> x8[kUnroll];
    int64_t at[kUnroll], row[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      at[u] = c0 + u * kThreads + threadIdx.x;
      row[u] = 0;
      int64_t col = at[u] * kVec;
      if (!flat && at[u] < total) {
        row[u] = at[u] / row_chunks;
        col = (at[u] - row[u] * row_chunks) * kVec;
      }
      x8[u] = at[u] < total ? load8(x + row[u] * ld_x + col) : zero8<T>();
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      uint32_t sc;
      const uint32_t c = quant8<T>(x8[u], sc);
      if (at[u] >= total) continue;
      codes[at[u]] = c;
      if ((at[u] & 3) == 0) scales[at[u] >> 2] = uint8_t(sc);
      if (out) {
        float v[kVec];
        values8(c, sc, v);
        const int64_t col = flat ? at[u] * kVec : (at[u] - row[u] * row_chunks) * kVec;
        store8(out + row[u] * ld_out + col, v);
      }
    }
  }
}

}  // namespace mx
}  // namespace dsa

using namespace dsa;

extern "C" int dsa_mxfp4_quant(const void* x, int x_type, int64_t ld_x, void* out, int64_t ld_out, uint8_t* codes,
                               uint8_t* scales, int64_t M, int64_t K, dsa_stream_t stream) {
  clear_error();
  DSA_CHECK_ARG(x && codes && scales, "mxfp4_quant: null x/codes/scales");
  DSA_CHECK_ARG(x_type == DSA_BF16 || x_type == DSA_FP16 || x_type == DSA_FP32, "mxfp4_quant: unknown x_type %d", x_type);
  DSA_CHECK_ARG(M >= 0 && K > 0 && K < (int64_t(1) << 31) && M <= (int64_t(1) << 40) / K, "mxfp4_quant: bad M/K");
  DSA_CHECK_ARG(K % mx::kBlock == 0, "mxfp4_quant: K=%lld not divisible by 32", (long long)K);
  const int es = x_type == DSA_FP32 ? 4 : 2;
  DSA_CHECK_ARG(ld_x >= K && ld_x * es % 16 == 0 && aligned(x, 16),
                "mxfp4_quant: x needs 16-byte alignment and a row stride >= K, a multiple of 16 bytes");
  DSA_CHECK_ARG(!out || (ld_out >= K && ld_out * es % 16 == 0 && aligned(out, 16)),
                "mxfp4_quant: out needs 16-byte alignment and a row stride >= K, a multiple of 16 bytes");
  DSA_CHECK_ARG(aligned(codes, 4), "mxfp4_quant: codes must be 4-byte aligned");
  if (M == 0) return DSA_OK;
  const int64_t total = M * (K / mx::kVec);
  const int per = mx::kThreads * mx::kUnroll;
  // one step of the loop a CTA up to 64 CTAs an SM: CTAs that come and go keep
  // loads and stores of the SM apart (32768 x 1024 fp32: 43.7 us, 6.55 TB/s,
  // against 48.1 with 8 CTAs an SM in step)
  const dim3 grid(unsigned(std::min<int64_t>((total + per - 1) / per, int64_t(num_sms()) * 64)));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  auto go = [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    return launch_pdl(mx::mxfp4_quant_kernel<T>, grid, dim3(mx::kThreads), 0, st, static_cast<const T*>(x), ld_x,
                      static_cast<T*>(out), ld_out, reinterpret_cast<uint32_t*>(codes), scales, total,
                      int(K / mx::kVec));
  };
  if (x_type == DSA_BF16)
    go(static_cast<__nv_bfloat16*>(nullptr));
  else if (x_type == DSA_FP16)
    go(static_cast<__half*>(nullptr));
  else
    go(static_cast<float*>(nullptr));
  DSA_CHECK_LAUNCH("mxfp4_quant");
  return DSA_OK;
}
