// The FP8 latent cache's write and read (record layout in kv_quant_dev.cuh).
//
// Write: per 64-dim block of the nope dims, with kv_window_write's
// arithmetic (inference.py:4578-4607 plus the e4m3 cast):
//   s = max(max |x|, 1e-4) * fl(1 / 448);  code = e4m3_rn(fl(x / s))
// The quotient is the correctly rounded one, from the correctly rounded
// reciprocal r of the block's s (one a lane) by Markstein's correction:
//   q = fl(x r), e = fl(q s - x), fl(q - e r)
// (in this sign a negative zero keeps its sign), two elements an instruction
// (a division each: 13.9 us for the 20,000 rows below, against 11.1 then).
// That it is holds because x is bf16: x has 128 significands and s = fl(m
// fl(1/448)) of a bf16 m 128 and the smallest scale's, and all 16,512 pairs come
// out right in exact arithmetic (Markstein's condition, q within an ulp, does
// not cover the 21 of them where e is rounded).  |x| >= 2^-10 s wherever the
// code is not zero and 2^-23 < s < 2^120, so nothing under- or overflows that
// the result shows.
// Read: bf16(float(code) * s), the rotary dims as they are.
// One warp a row, a lane 8 dims at a time: a block is 8 neighbouring lanes,
// so its maximum is three shuffles.  Both kernels are HBM streams (1024 B of
// bf16 on one side, a 608-B record on the other at 448 + 64 dims).  Measured:
// reading 132,000 selected records of 64 sequences 42.4 us, 5.36 TB/s (one row
// a warp at a time and 64-bit divisions for its place: 53.1); writing the
// 20,000 live rows of 8 padded sequences 10.2 us (the two rounds of a row's
// chunks fetched one after the other: 11.4; one or four rows a warp: 11.1,
// 11.8), about half of it two waves' latency of n_valid, pos and the row one
// after the other; one row each of 64 sequences 2.1 us.
#include "kv_quant_dev.cuh"

namespace dsa {
namespace kvq {

constexpr int kWarps = 8;
constexpr int kRows = 2;  // rows a warp has in flight
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

// the two bf16 of a 32-bit word, divided by s, as e4m3 codes (neg_r2: -r twice)
__device__ __forceinline__ uint32_t quotient_codes(uint32_t w, uint64_t neg_r2, uint64_t s2) {
  uint64_t nx, q, e;
  w ^= 0x80008000u;
  asm("mov.b64 %0, {%1, %2};" : "=l"(nx) : "r"(w << 16), "r"(w & 0xffff0000u));
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(q) : "l"(nx), "l"(neg_r2));
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(e) : "l"(q), "l"(s2), "l"(nx));
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(q) : "l"(e), "l"(neg_r2), "l"(q));
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(q));
  return __nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint64_t twice(float v) {
  uint64_t p;
  asm("mov.b64 %0, {%1, %1};" : "=l"(p) : "f"(v));
  return p;
}
__device__ __forceinline__ __nv_bfloat162 as_bf162(uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); }

// Sequences along y, groups of kRows tokens along x: a warp takes one group.
__global__ void __launch_bounds__(32 * kWarps) kv_quant_write_kernel(const WriteArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int n_chunks = a.nope / 8, all_chunks = n_chunks + a.rope / 8;
  const int used = a.nope + 2 * a.rope + 4 * (a.nope / kBlock);
  for (int b = blockIdx.y; b < a.B; b += gridDim.y) {
    const int n = a.n_valid ? min(a.n_valid[b], a.S) : a.S;
    const int64_t pos = a.pos[b];
    // the last win tokens (an earlier one's row belongs to a later one) at
    // positions >= 0
    const int64_t first = max(max(int64_t(n) - a.win, -pos), int64_t(0));
    for (int64_t s0 = first + (int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5)) * kRows; s0 < n;
         s0 += int64_t(gridDim.x) * kWarps * kRows) {
      const __nv_bfloat16* src = a.kv + b * a.ld_b + s0 * a.ld_s;
      uint8_t* dst[kRows];
#pragma unroll
      for (int u = 0; u < kRows; ++u)  // p < 2^32: a 32-bit position plus fewer than 2^31 tokens
        dst[u] = a.cache + b * a.bstride + (a.offset + uint32_t(pos + s0 + u) % uint32_t(a.win)) * a.rec;
      // the chunk count is not a multiple of 32 in general: whole warps take
      // part in the shuffles of a partly filled round
      uint4 raw[kRows], next[kRows];
      auto fetch = [&](int c) {
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
          next[u] = make_uint4(0, 0, 0, 0);
          if (c < all_chunks && s0 + u < n) next[u] = __ldg(reinterpret_cast<const uint4*>(src + u * a.ld_s) + c);
        }
      };
      fetch(lane);
      for (int c0 = 0; c0 < all_chunks; c0 += 32) {
        const int c = c0 + lane;
#pragma unroll
        for (int u = 0; u < kRows; ++u) raw[u] = next[u];
        fetch(c + 32);  // the next round's while this one is worked on
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
          // the block's maximum as bf16: a NaN stays
          __nv_bfloat162 m2 = __hmax2_nan(__hmax2_nan(__habs2(as_bf162(raw[u].x)), __habs2(as_bf162(raw[u].y))),
                                          __hmax2_nan(__habs2(as_bf162(raw[u].z)), __habs2(as_bf162(raw[u].w))));
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) m2 = __hmax2_nan(m2, __shfl_xor_sync(0xffffffffu, m2, o));
          const float m = __bfloat162float(__hmax_nan(m2.x, m2.y));
          if (s0 + u >= n) continue;  // (the warp's tokens: uniform)
          if (c < n_chunks) {
            const bool bad = !(m < INFINITY);
            const float sc = bad ? __uint_as_float(0x7fffffffu) : __fmul_rn(fmaxf(m, kEps), a.inv_max);
            uint32_t w[2] = {0u, 0u};
            if (!bad) {
              const uint64_t r2 = twice(-__frcp_rn(sc)), s2 = twice(sc);
              w[0] = quotient_codes(raw[u].x, r2, s2) | quotient_codes(raw[u].y, r2, s2) << 16;
              w[1] = quotient_codes(raw[u].z, r2, s2) | quotient_codes(raw[u].w, r2, s2) << 16;
            }
            *reinterpret_cast<uint2*>(dst[u] + 8 * c) = make_uint2(w[0], w[1]);
            if ((c & 7) == 0) reinterpret_cast<float*>(dst[u] + a.nope + 2 * a.rope)[c >> 3] = sc;
          } else if (c < all_chunks) {
            *reinterpret_cast<uint4*>(dst[u] + a.nope + 16 * (c - n_chunks)) = raw[u];
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kRows; ++u)
        if (s0 + u < n && 4 * lane < a.rec - used) *reinterpret_cast<uint32_t*>(dst[u] + used + 4 * lane) = 0u;
    }
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

// Sequences along y, groups of kReadRows output rows along x.
constexpr int kReadRows = 4;
template <bool kF32>
__global__ void __launch_bounds__(32 * kWarps) kv_quant_read_kernel(const ReadArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int n_chunks = a.nope / 8, all_chunks = n_chunks + a.rope / 8, D = a.nope + a.rope;
  for (int b = blockIdx.y; b < a.B; b += gridDim.y) {
    for (int64_t k0 = (int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5)) * kReadRows; k0 < a.K;
         k0 += int64_t(gridDim.x) * kWarps * kReadRows) {
      const uint8_t* src[kReadRows];  // NULL: a zero row
#pragma unroll
      for (int u = 0; u < kReadRows; ++u) {
        int64_t row = k0 + u;
        if (a.idx) {
          row = k0 + u < a.K ? a.idx[b * a.ld_idx + k0 + u] : -1;
          if (row >= a.rows) {
            if (a.status && lane == 0) atomicOr(a.status, 1);
            row = a.rows - 1;
          }
        }
        src[u] = row >= 0 && k0 + u < a.K ? a.cache + b * a.bstride + row * a.rec : nullptr;
      }
      for (int c = lane; c < all_chunks; c += 32) {
        const bool code = c < n_chunks;
        const int at = code ? 8 * c : a.nope + 16 * (c - n_chunks);
        const int at_s = code ? a.nope + 2 * a.rope + 4 * (c >> 3) : at + 8;
        uint2 lo[kReadRows], hi[kReadRows];  // codes and (in hi.x) their scale; or 16 B of rotary dims
#pragma unroll
        for (int u = 0; u < kReadRows; ++u) {
          lo[u] = hi[u] = make_uint2(0, 0);
          if (src[u]) {
            lo[u] = __ldg(reinterpret_cast<const uint2*>(src[u] + at));
            hi[u].x = __ldg(reinterpret_cast<const uint32_t*>(src[u] + at_s));
            if (!code) hi[u].y = __ldg(reinterpret_cast<const uint32_t*>(src[u] + at_s + 4));
          }
        }
#pragma unroll
        for (int u = 0; u < kReadRows; ++u) {
          if (k0 + u >= a.K) break;
          const int64_t t = int64_t(b) * a.K + k0 + u;
          float v[8];
          values8(lo[u], __uint_as_float(hi[u].x), v);
          const uint4 rope = make_uint4(lo[u].x, lo[u].y, hi[u].x, hi[u].y);
          if constexpr (kF32) {
            if (!code) bf16x8_to_f32(rope, v);
            float4* p = reinterpret_cast<float4*>(static_cast<float*>(a.out) + t * D) + 2 * c;
            p[0] = make_float4(v[0], v[1], v[2], v[3]);
            p[1] = make_float4(v[4], v[5], v[6], v[7]);
          } else {
            uint4 o = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                                 pack_bf16x2(v[6], v[7]));
            if (!code) o = rope;
            reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + t * D)[c] = o;
          }
        }
      }
    }
  }
}

// groups along x, sequences along y, at most ~16 CTAs an SM
static dim3 grid_for(int B, int64_t rows, int per_warp) {
  const int64_t x = (rows + kWarps * per_warp - 1) / (kWarps * per_warp);
  const int64_t most = int64_t(num_sms()) * 16;
  const int64_t y = std::min<int64_t>(B, 65535);
  return dim3(unsigned(std::min(x, std::max<int64_t>(1, most / y))), unsigned(y));
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
  DSA_CHECK_ARG(S >= 0 && win > 0 && offset >= 0 && win <= cache_rows && offset <= cache_rows - win,
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
  launch_pdl(kvq::kv_quant_write_kernel, kvq::grid_for(B, std::min(S, win), kvq::kRows), dim3(32 * kvq::kWarps), 0, reinterpret_cast<cudaStream_t>(stream), a);
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
  auto k = out_f32 ? kvq::kv_quant_read_kernel<true> : kvq::kv_quant_read_kernel<false>;
  launch_pdl(k, kvq::grid_for(B, K, kvq::kReadRows), dim3(32 * kvq::kWarps), 0, reinterpret_cast<cudaStream_t>(stream), a);
  DSA_CHECK_LAUNCH("kv_quant_read");
  return DSA_OK;
}
