// MXFP4 quantisation of a matrix along its rows (formulas in mxfp4_dev.cuh).
//
// 16-bit inputs: a lane holds 16 elements, two lanes a block of 32, so the
// block's maximum is one shuffle; the two take turns eight by eight (0-7 and
// 16-23, 8-15 and 24-31), so that neighbouring lanes read and write
// neighbouring bytes.  fp32: 8 elements a lane and two blocks in flight (32768
// x 1024 with values: 43.7 us against 46.3).  Nothing touches shared memory.  The kernel is
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
template <typename T>
struct Shape {
  static constexpr int H = sizeof(T) == 2 ? 2 : 1;  // eights a lane
  static constexpr int kLanes = 4 / H;              // lanes a block
  static constexpr int kUnroll = 2 / H;             // blocks a lane has in flight
};

// Eight elements by plain loads: out may be x, so x is neither __restrict__ nor
// read through the non-coherent path.  A block's loads all precede its stores
// (its maximum is exchanged between them), and no other block's elements lie
// in its place.
template <typename T>
__device__ __forceinline__ Vec8<T> load8_plain(const T* p) {
  Vec8<T> r;
#pragma unroll
  for (int i = 0; i < int(sizeof(T) / 2); ++i) r.w[i] = reinterpret_cast<const uint4*>(p)[i];
  return r;
}

// Blocks [0, blocks) in row order; the codes and scales are contiguous, x and
// out have row strides.
template <typename T>
__global__ void __launch_bounds__(kThreads) mxfp4_quant_kernel(const T* x, int64_t ld_x, T* out, int64_t ld_out,
                                                               uint32_t* __restrict__ codes,
                                                               uint8_t* __restrict__ scales, int64_t blocks,
                                                               int row_blocks) {
  using S = Shape<T>;
  constexpr int kPer = kThreads / S::kLanes;  // blocks a CTA takes at a time
  pdl_wait();
  pdl_launch_dependents();
  const bool flat = ld_x == int64_t(row_blocks) * kBlock && (!out || ld_out == ld_x);
  const int part = threadIdx.x % S::kLanes;
  // whole warps stay in the loop: the block maximum is a warp shuffle
  for (int64_t c0 = int64_t(blockIdx.x) * kPer * S::kUnroll; c0 < blocks; c0 += int64_t(gridDim.x) * kPer * S::kUnroll) {
    Vec8<T> v[S::kUnroll][S::H];
    int64_t row[S::kUnroll], col[S::kUnroll];
#pragma unroll
    for (int u = 0; u < S::kUnroll; ++u) {
      const int64_t at = c0 + u * kPer + threadIdx.x / S::kLanes;
      row[u] = 0;
      col[u] = at * kBlock;
      if (!flat && at < blocks) {
        row[u] = at / row_blocks;
        col[u] = (at - row[u] * row_blocks) * kBlock;
      }
#pragma unroll
      for (int h = 0; h < S::H; ++h)
        v[u][h] = at < blocks ? load8_plain(x + row[u] * ld_x + col[u] + (h * S::kLanes + part) * kVec) : zero8<T>();
    }
#pragma unroll
    for (int u = 0; u < S::kUnroll; ++u) {
      const int64_t at = c0 + u * kPer + threadIdx.x / S::kLanes;
      uint32_t sc, c[S::H];
      quant(v[u], sc, c);
      if (at >= blocks) continue;
      if (part == 0) scales[at] = uint8_t(sc);
#pragma unroll
      for (int h = 0; h < S::H; ++h) {
        const int e = h * S::kLanes + part;  // the lane's eight of the block
        codes[4 * at + e] = c[h];
        if (out) {
          float f[kVec];
          values8(c[h], sc, f);
          store8(out + row[u] * ld_out + col[u] + e * kVec, f);
        }
      }
    }
  }
}

}  // namespace mx
}  // namespace dsa

using namespace dsa;

// out [M rows of `row` bytes, `pitch_o` apart] shares memory with x (`pitch_x`),
// other than being x, or a block of columns of the same rows beside x's
static bool partly_covers(const void* x, const void* out, int64_t pitch_x, int64_t pitch_o, int64_t row, int64_t M) {
  const auto a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(out);
  if (M == 0 || (a == b && (M == 1 || pitch_x == pitch_o))) return false;
  if (a + (M - 1) * pitch_x + row <= b || b + (M - 1) * pitch_o + row <= a) return false;
  if (pitch_x != pitch_o) return true;
  const int64_t d = int64_t((a > b ? a - b : b - a) % uintptr_t(pitch_x));
  return d < row || pitch_x - d < row;
}

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
  DSA_CHECK_ARG(!out || !partly_covers(x, out, ld_x * es, ld_out * es, K * es, M),
                "mxfp4_quant: out may be x or lie beside it, not overlap it");
  DSA_CHECK_ARG(aligned(codes, 4), "mxfp4_quant: codes must be 4-byte aligned");
  if (M == 0) return DSA_OK;
  const int64_t blocks = M * (K / mx::kBlock);
  const int per = mx::kThreads / 2;  // of either shape, blocks a CTA has in flight
  // one step of the loop a CTA up to 64 CTAs an SM: CTAs that come and go keep
  // loads and stores of the SM apart (32768 x 1024 fp32: 43.7 us, 6.55 TB/s,
  // against 48.1 with 8 CTAs an SM in step)
  const dim3 grid(unsigned(std::min<int64_t>((blocks + per - 1) / per, int64_t(num_sms()) * 64)));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  auto go = [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    return launch_pdl(mx::mxfp4_quant_kernel<T>, grid, dim3(mx::kThreads), 0, st, static_cast<const T*>(x), ld_x,
                      static_cast<T*>(out), ld_out, reinterpret_cast<uint32_t*>(codes), scales, blocks,
                      int(K / mx::kBlock));
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
