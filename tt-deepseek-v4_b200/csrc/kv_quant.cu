// The FP8 latent cache's write and read (record layout in kv_quant_dev.cuh).
//
// Write: per 64-dim block of the nope dims, with kv_window_write's
// arithmetic (inference.py:4578-4607 plus the e4m3 cast):
//   s = max(max |x|, 1e-4) * fl(1 / 448);  code = e4m3_rn(x / s)  (IEEE div)
// Read: bf16(float(code) * s), the rotary dims as they are.
// One warp a row, a lane 8 dims at a time: a block is 8 neighbouring lanes,
// so its maximum is three shuffles.  Both kernels are HBM streams (1024 B of
// bf16 on one side, a 608-B record on the other at 448 + 64 dims).
#include "kv_quant_dev.cuh"

namespace dsa {
namespace kvq {

constexpr int kWarps = 8;
constexpr float kFp8Max = 448.f;
constexpr float kEps = 1e-4f;

struct WriteArgs {
  const __nv_bfloat16* kv;
  int64_t ld_b, ld_s;        // elements
  uint8_t* cache;
  int64_t bstride;           // bytes
  const int32_t* pos;
  const int32_t* n_valid;    // tokens of each sequence (may be NULL: all S)
  int B, S, nope, rope, rec;
  int win;
  int64_t offset;
  float inv_max;
};

__global__ void __launch_bounds__(32 * kWarps) kv_quant_write_kernel(const WriteArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t n_tok = int64_t(a.B) * a.S;
  const int n_chunks = a.nope / 8, all_chunks = n_chunks + a.rope / 8;
  for (int64_t t = int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5); t < n_tok; t += int64_t(gridDim.x) * kWarps) {
    const int b = int(t / a.S), s = int(t - int64_t(b) * a.S);
    const int n = a.n_valid ? min(a.n_valid[b], a.S) : a.S;
    // the last win tokens: an earlier one's row belongs to a later one
    if (s >= n || s < n - a.win) continue;
    const int64_t p = int64_t(a.pos[b]) + s;
    if (p < 0) continue;
    const __nv_bfloat16* src = a.kv + b * a.ld_b + s * a.ld_s;
    // p < 2^32: a 32-bit position plus fewer than 2^31 tokens
    uint8_t* dst = a.cache + b * a.bstride + (a.offset + uint32_t(p) % uint32_t(a.win)) * a.rec;
    float* dst_scales = reinterpret_cast<float*>(dst + a.nope + 2 * a.rope);
    // the chunk count is not a multiple of 32 in general: whole warps take
    // part in the shuffles of a partly filled round
    for (int c0 = 0; c0 < all_chunks; c0 += 32) {
      const int c = c0 + lane;
      uint4 raw = make_uint4(0, 0, 0, 0);
      if (c < all_chunks) raw = __ldg(reinterpret_cast<const uint4*>(src) + c);
      float v[8];
      bf16x8_to_f32(raw, v);
      uint32_t m = 0;  // fp32 bits order as integers, NaN and infinity on top
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      if (c < n_chunks) {
        const bool bad = m >= 0x7f800000u;
        const float sc = bad ? __uint_as_float(0x7fffffffu) : __fmul_rn(fmaxf(__uint_as_float(m), kEps), a.inv_max);
        uint32_t w[2] = {0u, 0u};
        if (!bad) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const __nv_fp8x2_storage_t q = __nv_cvt_float2_to_fp8x2(
                make_float2(__fdiv_rn(v[2 * i], sc), __fdiv_rn(v[2 * i + 1], sc)), __NV_SATFINITE, __NV_E4M3);
            w[i >> 1] |= uint32_t(q) << (16 * (i & 1));
          }
        }
        *reinterpret_cast<uint2*>(dst + 8 * c) = make_uint2(w[0], w[1]);
        if ((c & 7) == 0) dst_scales[c >> 3] = sc;
      } else if (c < all_chunks) {
        *reinterpret_cast<uint4*>(dst + a.nope + 16 * (c - n_chunks)) = raw;
      }
    }
    const int used = a.nope + 2 * a.rope + 4 * (a.nope / kBlock);
    if (4 * lane < a.rec - used) *reinterpret_cast<uint32_t*>(dst + used + 4 * lane) = 0u;
  }
}

struct ReadArgs {
  const uint8_t* cache;
  int64_t bstride, rows;
  const int32_t* idx;  // NULL: row k of the output is cache row k
  int64_t ld_idx;
  void* out;
  int64_t K;
  int B, nope, rope, rec;
  int32_t* status;
};

template <bool kF32>
__global__ void __launch_bounds__(32 * kWarps) kv_quant_read_kernel(const ReadArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t n_rows = int64_t(a.B) * a.K;
  const int n_chunks = a.nope / 8, all_chunks = n_chunks + a.rope / 8;
  for (int64_t t = int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5); t < n_rows; t += int64_t(gridDim.x) * kWarps) {
    const int64_t b = t / a.K, k = t - b * a.K;
    int64_t row = k;
    if (a.idx) {
      row = a.idx[b * a.ld_idx + k];
      if (row >= a.rows) {
        if (a.status && lane == 0) atomicOr(a.status, 1);
        row = a.rows - 1;
      }
    }
    const bool ok = row >= 0;
    const uint8_t* src = a.cache + b * a.bstride + (ok ? row : 0) * a.rec;
    const float* scales = reinterpret_cast<const float*>(src + a.nope + 2 * a.rope);
    for (int c = lane; c < all_chunks; c += 32) {
      uint4 o = make_uint4(0, 0, 0, 0);
      float v[8];
      if (c < n_chunks) {
        if (ok) {
          values8(__ldg(reinterpret_cast<const uint2*>(src) + c), __ldg(scales + (c >> 3)), v);
          o = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                         pack_bf16x2(v[6], v[7]));
        }
      } else if (ok) {
        o = __ldg(reinterpret_cast<const uint4*>(src + a.nope) + (c - n_chunks));
      }
      if constexpr (kF32) {
        if (c >= n_chunks || !ok) bf16x8_to_f32(o, v);
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(a.out) + t * (a.nope + a.rope)) + 2 * c;
        p[0] = make_float4(v[0], v[1], v[2], v[3]);
        p[1] = make_float4(v[4], v[5], v[6], v[7]);
      } else {
        reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + t * (a.nope + a.rope))[c] = o;
      }
    }
  }
}

static int check_row(const char* what, const void* cache, int64_t bstride, int64_t rows, int B, int D, int rope_dim) {
  DSA_CHECK_ARG(D > 0 && D <= 8192 && rope_dim >= 0 && rope_dim < D && rope_dim % 8 == 0 && (D - rope_dim) % kBlock == 0,
                "%s: D - rope_dim must be a positive multiple of 64, rope_dim a multiple of 8, D <= 8192", what);
  DSA_CHECK_ARG(B >= 0 && rows > 0 && rows <= INT32_MAX, "%s: bad B/rows", what);
  DSA_CHECK_ARG(aligned(cache, 16) && bstride % 16 == 0 && (B <= 1 || bstride >= rows * row_bytes(D - rope_dim, rope_dim)),
                "%s: the cache needs 16-byte alignment and a batch stride that covers its rows", what);
  return DSA_OK;
}

}  // namespace kvq
}  // namespace dsa

using namespace dsa;

extern "C" size_t dsa_kv_quant_row_bytes(int D, int rope_dim) {
  if (D <= 0 || D > 8192 || rope_dim < 0 || rope_dim >= D || rope_dim % 8 || (D - rope_dim) % kvq::kBlock) return 0;
  return size_t(kvq::row_bytes(D - rope_dim, rope_dim));
}

extern "C" int dsa_kv_quant_write(const void* kv, int64_t ld_b, int64_t ld_s, void* cache, int64_t cache_bstride,
                                  int64_t cache_rows, const int32_t* pos, const int32_t* n_valid, int B, int S, int D,
                                  int rope_dim, int win, int64_t offset, dsa_stream_t stream) {
  clear_error();
  DSA_CHECK_ARG(kv && cache && pos, "kv_quant_write: null kv/cache/pos");
  const int rc = kvq::check_row("kv_quant_write", cache, cache_bstride, cache_rows, B, D, rope_dim);
  if (rc) return rc;
  DSA_CHECK_ARG(S >= 0 && win > 0 && offset >= 0 && offset + win <= cache_rows,
                "kv_quant_write: the ring's rows [offset, offset + win) must lie in the cache");
  DSA_CHECK_ARG(aligned(kv, 16) && ld_b % 8 == 0 && ld_s % 8 == 0,
                "kv_quant_write: kv needs 16-byte alignment and strides that are multiples of 8 elements");
  if (B == 0 || S == 0) return DSA_OK;
  kvq::WriteArgs a{};
  a.kv = static_cast<const __nv_bfloat16*>(kv);
  a.ld_b = ld_b;
  a.ld_s = ld_s;
  a.cache = static_cast<uint8_t*>(cache);
  a.bstride = cache_bstride;
  a.pos = pos;
  a.n_valid = n_valid;
  a.B = B;
  a.S = S;
  a.nope = D - rope_dim;
  a.rope = rope_dim;
  a.rec = kvq::row_bytes(a.nope, a.rope);
  a.win = win;
  a.offset = offset;
  a.inv_max = float(1.0 / double(kvq::kFp8Max));  // rounded once, as the reference's constant
  const int64_t n_tok = int64_t(B) * S;
  const dim3 grid(unsigned(std::min<int64_t>((n_tok + kvq::kWarps - 1) / kvq::kWarps, int64_t(num_sms()) * 32)));
  launch_pdl(kvq::kv_quant_write_kernel, grid, dim3(32 * kvq::kWarps), 0, reinterpret_cast<cudaStream_t>(stream), a);
  DSA_CHECK_LAUNCH("kv_quant_write");
  return DSA_OK;
}

extern "C" int dsa_kv_quant_read(const void* cache, int64_t cache_bstride, int64_t cache_rows, const int32_t* idx,
                                 int64_t ld_idx, void* out, int out_f32, int B, int64_t K, int D, int rope_dim,
                                 int32_t* status, dsa_stream_t stream) {
  clear_error();
  DSA_CHECK_ARG(cache && out, "kv_quant_read: null cache/out");
  const int rc = kvq::check_row("kv_quant_read", cache, cache_bstride, cache_rows, B, D, rope_dim);
  if (rc) return rc;
  DSA_CHECK_ARG(K >= 0 && K <= INT32_MAX, "kv_quant_read: bad K");
  DSA_CHECK_ARG(idx ? (B <= 1 || ld_idx >= K) : K <= cache_rows,
                "kv_quant_read: ld_idx < K, or more rows than the cache holds");
  DSA_CHECK_ARG(aligned(out, 16), "kv_quant_read: out must be 16-byte aligned");
  if (B == 0 || K == 0) return DSA_OK;
  kvq::ReadArgs a{};
  a.cache = static_cast<const uint8_t*>(cache);
  a.bstride = cache_bstride;
  a.rows = cache_rows;
  a.idx = idx;
  a.ld_idx = ld_idx;
  a.out = out;
  a.K = K;
  a.B = B;
  a.nope = D - rope_dim;
  a.rope = rope_dim;
  a.rec = kvq::row_bytes(a.nope, a.rope);
  a.status = status;
  const int64_t n_rows = int64_t(B) * K;
  const dim3 grid(unsigned(std::min<int64_t>((n_rows + kvq::kWarps - 1) / kvq::kWarps, int64_t(num_sms()) * 32)));
  auto k = out_f32 ? kvq::kv_quant_read_kernel<true> : kvq::kv_quant_read_kernel<false>;
  launch_pdl(k, grid, dim3(32 * kvq::kWarps), 0, reinterpret_cast<cudaStream_t>(stream), a);
  DSA_CHECK_LAUNCH("kv_quant_read");
  return DSA_OK;
}
