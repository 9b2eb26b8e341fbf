// Projections over MXFP4 weights on the tcgen05 tensor cores:
//   Y[b, n] = sum_k q(X)[b, k] * W[n, k],   b < B, n < N
// with W in MXFP4 and X quantised to MXFP4 in the call (mxfp4_dev.cuh); sums
// in fp32, Y bf16 or fp32.  kind::mxf4 multiplies the 4-bit elements and the
// block scales in the tensor cores: products of E2M1 values are exact and no
// operand is expanded.
//
// Two launches: X's quantisation into tiles of the weight's layout, then the
// product, whose weight loads start before the first has ended.  Where a CTA's
// share of X is a few rows (kFuse), one launch: the epilogue's warps, idle
// until the first sum, quantise it into shared memory themselves.
//
// Weight layout (dsa_linear_mxfp4_pack, once at load time): per (128-row tile
// t, 256-wide k-block kb) 17 KB: the codes of the 128 rows as a 128-byte
// swizzled K-major operand (row r at r * 128 B, 16-byte chunk c at
// (c ^ (r & 7)) * 16), then their 8 scales a row as two 512-byte blocks of
// four (byte (r % 32) * 16 + (r / 32) * 4 + j), zero past N and K.  A CTA's
// k-range is one contiguous run of memory that it reads with 17 KB bulk copies.
//
// X's scratch holds the same tiles with Bt token rows: codes, then 1 KB of
// scales for each 128 tokens.
//
// A work item is (128 weight rows, Bt <= 192 tokens):
//   warp 0      producer: per k-block two bulk copies, a weight tile and an X
//               tile, into a ring;
//   warp 6      scales from shared into tensor memory (tcgen05.cp), a set of
//               columns for each stage of the ring;
//   warp 1      MMA issuer: Y^T = W . X^T, M = 128 weight rows, N = Bt
//               tokens, K = 64 a step, into one of two accumulators: the
//               epilogue of item i overlaps item i + 1;
//   warps 2-5   epilogue, thread = weight row: rounding, a staging tile and a
//               TMA store (element stores where Y's rows are not 16-byte
//               aligned).
// One thread issued copies of scales and products at first: a tcgen05.cp
// costs its issuer ~100 cycles, so a k-block took 1400 cycles against ~400 of
// MMA time (the product of 4096 x 4096 x 8192: 128 us).  Now a k-block of 192
// tokens takes ~630, what shared memory moves in that time: 44 KB written by
// the copies and 40 KB read by the four products at 128 B a cycle.
// Measured whole: 4096 x 4096 x 8192 80.3 us in bursts (3.4 PFLOP/s; x's
// quantisation ~15 of them; 88-91 back to back, under the power cap), 64 x 32768
// x 1024 7.7 us (2.9 TB/s), 1 x 1024 x 4096 4.85 us.
// Tensor memory: 2 x 192 accumulator columns, 128 of scales (8 a stage for W, 8
// for each 128 tokens of X).
//
// Few items (decode): the C CTAs of a cluster share an item, each over its
// own part of K.  After the last product a cluster barrier frees every ring;
// each CTA writes its partial [Bt][128] there, copies each owner's rows to it
// through distributed shared memory, and the owner sums the C partials in rank
// order: the same sum on every run.
//
// Every wait is bounded.  One that runs out sets a status bit and its CTA's
// abort flag, at which the CTA's other waits return unless their phase is over:
// its roles issue and store nothing more, what is in flight lands, and the CTA
// leaves through the same barriers as ever.  Its tiles stay unwritten; a split
// item's other owners get NaN from it.  (0-3 % of the times below: 64 x 32768 x 1024
// 7.4 -> 7.7 us, 1024 x 4096 x 8192 27.8 -> 28.0.)
#include "cluster.cuh"
#include "common.cuh"
#include "mxfp4_dev.cuh"
#include "tc05.cuh"
#include "tma.cuh"

#include <algorithm>
#include <cstring>
#include <mutex>
#include <type_traits>

namespace dsa {
namespace lmx {

constexpr int TILE_N = 128;
constexpr int KBW = 256;                        // k a stage: 128 B of codes a row
constexpr int kSfPerKb = KBW / mx::kBlock;      // 8 scales
constexpr int kCodeBytes = TILE_N * KBW / 2;    // 16 KB
constexpr int kSfBytes = TILE_N * kSfPerKb;     // 1 KB for each 128 rows
constexpr int kWBytes = kCodeBytes + kSfBytes;  // a weight tile
constexpr int kMaxBt = 192;
constexpr int kMaxStages = 8;
constexpr int kMaxSplit = 16;
constexpr int THREADS = 224;
constexpr int kSmemBytes = 232448;
constexpr int kAuxBytes = 512;
constexpr int kFuseUnits = 32;                  // (token, k-block) units of X a CTA quantises itself, at most
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColSf = 2 * kMaxBt;         // scales of each stage: 8 columns of W, 8 a group of X
__host__ __device__ constexpr int sf_cols(int groups) { return 8 + 8 * groups; }
__host__ __device__ constexpr int max_stages(int groups) {
  return (int(kTmemCols) - int(kColSf)) / sf_cols(groups) < kMaxStages ? (int(kTmemCols) - int(kColSf)) / sf_cols(groups)
                                                                       : kMaxStages;
}
static_assert(kWBytes % 1024 == 0, "the swizzled operands start on 1024 B");

struct Args {
  const uint8_t* w;
  const uint8_t* x;     // X's tiles [m tile][k-block]; kFuse: X itself
  int64_t ld_x;         // kFuse: X's row stride, type and columns
  int x_type, K;
  void* y;
  int64_t ld_y;
  int B, Bt, groups, N, nkb, n_tiles, m_tiles;
  int split, rows_per;  // C CTAs an item; token rows each of them finishes
  int n_stages, tma_store;
  uint32_t stage_bytes, half_bytes, x_off, part_off, recv_off, out_off, aux_off;
  int32_t* status;
  long long wait_limit;
};

struct Aux {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t sf_full[kMaxStages];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint64_t ready;
  uint64_t x_full;
  uint64_t drained;    // gave up: the loads have landed, both issuers' work is done
  uint32_t tmem_base;
  int abort;
  int issued;          // stages whose loads were requested
};
static_assert(sizeof(Aux) <= kAuxBytes, "aux block");

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(src), "r"(x), "r"(y)
               : "memory");
}

// A phase's end, or false once the CTA has given up.  The loop lies inline only
// in the fused kernel, whose few waits mostly begin before their phase's end
// (inline / called: 8 x 1024 x 4096 5.47 / 5.60 us); inline everywhere, a
// k-block of the ring takes 20 cycles more (1024 x 4096 x 8192: 28.8 / 27.9).
__device__ __forceinline__ bool wait_loop(uint32_t bar, uint32_t parity, volatile int* abort, int32_t* status,
                                          long long limit) {
  const long long t0 = clock64();
  for (;;) {
    if (tc::mbar_try_wait(bar, parity)) return true;
    if (*abort) return false;
    if (clock64() - t0 > limit) {
      if (status) atomicOr(status, 2);
      *abort = 1;
      return false;
    }
  }
}
__device__ __noinline__ bool wait_called(uint32_t bar, uint32_t parity, volatile int* abort, int32_t* status,
                                         long long limit) {
  return wait_loop(bar, parity, abort, status, limit);
}

// Warps 0, 1 and 6 of a CTA that gave up, once its roles have ended: `drained`
// completes when its loads have landed and its tensor core work is done.  (A
// limit of its own: the caller's may be too short for any of it.)
__device__ __noinline__ void drain(Aux* aux, int n_stages, int32_t* status) {
  if (threadIdx.x == 0) {
    const int n = aux->issued;
    for (int i = max(0, n - n_stages); i < n; ++i)
      tc::mbar_wait(smem_u32(&aux->full[i % n_stages]), (i / n_stages) & 1, status, 2);
    tc::mbar_arrive(smem_u32(&aux->drained));
  } else if (threadIdx.x >= 32 && tc::elect_one()) {
    tc::mma_commit(smem_u32(&aux->drained));
  }
  __syncwarp();
  tc::mbar_wait(smem_u32(&aux->drained), 0, status, 2);
}

// The partial of a thread whose sums never came, once nothing else writes there
__device__ __noinline__ void poison(float* column, int rows, const uint64_t* drained, int32_t* status) {
  tc::mbar_wait(smem_u32(drained), 0, status, 2);
  for (int i = 0; i < rows; ++i) column[i * TILE_N] = __uint_as_float(0x7fffffffu);
}

template <bool kF32>
using OutT = typename std::conditional<kF32, float, __nv_bfloat16>::type;
template <bool kF32>
__device__ __forceinline__ OutT<kF32> to_out(float v) {
  if constexpr (kF32) return v;
  else return f2bf(v);
}

// Staging of a finished tile for the TMA store.  bf16: two halves of 64
// columns, [row][128 B] with the 128-byte swizzle (what stmatrix and the
// store take without bank conflicts); fp32: [row][128].
template <bool kF32>
__device__ __forceinline__ OutT<kF32>* stage_at(uint8_t* stage, uint32_t half_bytes, int row, int n) {
  if constexpr (kF32) return reinterpret_cast<float*>(stage) + row * TILE_N + n;
  else
    return reinterpret_cast<__nv_bfloat16*>(stage + (n >> 6) * half_bytes + row * 128 +
                                            ((((n >> 3) & 7) ^ (row & 7)) << 4)) + (n & 7);
}

// the staged tile's rows to Y[b0.., 128 t ..] (one thread)
template <bool kF32>
__device__ __forceinline__ void store_tile(const CUtensorMap* tm_y, uint32_t stage, uint32_t half_bytes, int t, int b0,
                                           int N) {
  if constexpr (kF32) {
    tma_store_2d(tm_y, stage, t * TILE_N, b0);
  } else {
    tma_store_2d(tm_y, stage, t * TILE_N, b0);
    if (t * TILE_N + 64 < N) tma_store_2d(tm_y, stage + half_bytes, t * TILE_N + 64, b0);
  }
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

// CNT values of this thread's weight row, token rows [row, ..), to Y
template <bool kF32, int CNT>
__device__ __forceinline__ void store_rows(const Args& a, int64_t row, int rows, int n, const float* v) {
  if (n >= a.N) return;
  OutT<kF32>* o = static_cast<OutT<kF32>*>(a.y) + row * a.ld_y + n;
  if (rows >= CNT) {  // no guard inside: the stores leave back to back
#pragma unroll
    for (int i = 0; i < CNT; ++i) o[i * a.ld_y] = to_out<kF32>(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < CNT; ++i)
      if (i < rows) o[i * a.ld_y] = to_out<kF32>(v[i]);
  }
}

// A k-block of one token on a half warp, 16 elements a lane (past K: zeros)
template <typename T>
struct KBlock {
  mx::Vec8<T> h[2];
};
template <typename T>
__device__ __forceinline__ KBlock<T> load_kblock(const T* row, int kb, int K, int lane, bool ok) {
  KBlock<T> x;
  const int k = kb * KBW + (lane & 15) * 2 * mx::kVec;
#pragma unroll
  for (int h = 0; h < 2; ++h)
    x.h[h] = ok && k + h * mx::kVec < K ? mx::load8(row + k + h * mx::kVec) : mx::zero8<T>();
  return x;
}

// ... quantised into row r of a tile of Bt rows: the row's codes and its eight
// scales (the whole warp calls it; a half with ok false stores nothing)
template <typename T>
__device__ __forceinline__ void put_kblock(uint8_t* tile, const KBlock<T>& x, int Bt, int r, int lane, bool ok) {
  uint32_t sc;
  uint32_t c[2];
  mx::quant(x.h, sc, c);
  if (!ok) return;
  const int l = lane & 15;
  *reinterpret_cast<uint2*>(tile + r * 128 + (((l >> 1) ^ (r & 7)) << 4) + (l & 1) * 8) = make_uint2(c[0], c[1]);
  if ((l & 1) == 0)
    tile[Bt * (KBW / 2) + (r >> 7) * kSfBytes + (l >> 3) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4 + ((l >> 1) & 3)] =
        uint8_t(sc);
}

// kFuse: the CTA's k-blocks [kb0, kb1) of every token into its tiles at xs, a
// half warp (of 8) a (k-block, token) unit, two units in flight
template <typename T>
__device__ __forceinline__ void fill_x(const Args& a, uint8_t* xs, uint32_t x_tile, int kb0, int kb1, int w, int lane) {
  const T* x = reinterpret_cast<const T*>(a.x);
  const int units = (kb1 - kb0) * a.B;
  constexpr int kFly = 2;
  for (int u0 = 2 * w; u0 < units; u0 += 8 * kFly) {
    KBlock<T> v[kFly];
    int kb[kFly], b[kFly];
    bool ok[kFly];
#pragma unroll
    for (int i = 0; i < kFly; ++i) {
      const int u = u0 + (lane >> 4) + 8 * i;
      ok[i] = u < units;
      kb[i] = u / a.B;
      b[i] = u - kb[i] * a.B;
      v[i] = load_kblock(x + b[i] * a.ld_x, kb0 + kb[i], a.K, lane, ok[i]);
    }
#pragma unroll
    for (int i = 0; i < kFly; ++i) put_kblock<T>(xs + kb[i] * x_tile, v[i], a.Bt, b[i], lane, ok[i]);
  }
}

template <bool kF32, bool kFuse>
__global__ void __launch_bounds__(THREADS, 1) linear_mxfp4_kernel(const Args a,
                                                                  const __grid_constant__ CUtensorMap tm_y) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Aux* aux = reinterpret_cast<Aux*>(smem + a.aux_off);
  const uint32_t sbase = smem_u32(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int C = a.split;
  const int rank = C > 1 ? int(lin::cluster_rank()) : 0;
  const int cid = blockIdx.x / C, n_cl = gridDim.x / C;
  const int n_items = a.n_tiles * a.m_tiles;
  const int kb0 = rank * a.nkb / C, kb1 = (rank + 1) * a.nkb / C;
  const int NS = a.n_stages;
  const uint32_t x_bytes = uint32_t(a.Bt) * (KBW / 2);
  const uint32_t x_tile = x_bytes + uint32_t(a.groups) * kSfBytes;
  const uint32_t stage_tx = kFuse ? kWBytes : kWBytes + x_tile;

  if (warp == 1) {
    tc::tmem_alloc(smem_u32(&aux->tmem_base), kTmemCols);
    tc::tmem_relinquish();
  }
  if (tid == 0) {
    for (int s = 0; s < NS; ++s) {
      tc::mbar_init(smem_u32(&aux->full[s]), 1);
      tc::mbar_init(smem_u32(&aux->empty[s]), 1);
      tc::mbar_init(smem_u32(&aux->sf_full[s]), 1);
    }
    for (int s = 0; s < 2; ++s) {
      tc::mbar_init(smem_u32(&aux->acc_full[s]), 1);
      tc::mbar_init(smem_u32(&aux->acc_empty[s]), 4);
    }
    tc::mbar_init(smem_u32(&aux->x_full), 4);
    tc::mbar_init(smem_u32(&aux->ready), 1);  // the owner's arrival + the copied bytes
    tc::mbar_init(smem_u32(&aux->drained), 3);
    aux->abort = 0;
    tc::mbar_fence_init();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = aux->tmem_base;

  // The weights' first tiles are requested before the dependency wait: the
  // kernel before this one is x's quantisation, which let it start only after
  // its own wait, so whatever wrote the weights has completed.  kFuse: the
  // kernel before may be the one that packed them.
  if constexpr (kFuse) pdl_wait();
  int npre = 0;
  if (warp == 0 && lane == 0) {
    for (int item = cid; item < n_items && npre < NS; item += n_cl) {
      const uint8_t* wt = a.w + (int64_t(item / a.m_tiles) * a.nkb + kb0) * kWBytes;
      for (int kb = kb0; kb < kb1 && npre < NS; ++kb, ++npre, wt += kWBytes) {
        const uint32_t fb = smem_u32(&aux->full[npre]);
        tma::mbar_arrive_expect_tx(fb, stage_tx);
        lin::bulk_load(sbase + npre * a.stage_bytes, wt, kWBytes, fb);
      }
    }
  }
  if constexpr (!kFuse) pdl_wait();
  pdl_launch_dependents();

  auto wait = [&](const uint64_t* bar, uint32_t parity) {
    const uint32_t at = smem_u32(bar);
    if (tc::mbar_try_wait(at, parity)) return true;
    if constexpr (kFuse) return wait_loop(at, parity, &aux->abort, a.status, a.wait_limit);
    else return wait_called(at, parity, &aux->abort, a.status, a.wait_limit);
  };
  // The issuers run their loops to the end whatever becomes of a wait: `go`
  // of the elected lane, which issues, says whether it still does, and a lane
  // that has given up waits no more.  (A vote and an exit a k-block cost 40
  // cycles of 630.)
  // a stage's address, barrier and parity advance by counters: a division a
  // k-block showed in the issuers' time
  if (warp == 0) {
    // ---------------------------------------------------------------- producer
    if (lane == 0) {
      int it = 0, s = 0;
      uint32_t ph = 1;  // parity of the stage's last release
      bool go = true;
      for (int item = cid; go && item < n_items; item += n_cl) {
        const int t = item / a.m_tiles, mt = item - t * a.m_tiles;
        const uint8_t* wt = a.w + (int64_t(t) * a.nkb + kb0) * kWBytes;
        const uint8_t* xt = a.x + (int64_t(mt) * a.nkb + kb0) * x_tile;
        for (int kb = kb0; kb < kb1; ++kb, ++it, wt += kWBytes, xt += x_tile) {
          const uint32_t st = sbase + s * a.stage_bytes;
          const uint32_t fb = smem_u32(&aux->full[s]);
          if (it >= npre) {
            if (it >= NS && !wait(&aux->empty[s], ph)) {
              go = false;
              break;
            }
            tma::mbar_arrive_expect_tx(fb, stage_tx);
            lin::bulk_load(st, wt, kWBytes, fb);
          }
          if constexpr (!kFuse) lin::bulk_load(st + kWBytes, xt, x_tile, fb);
          if (++s == NS) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      aux->issued = it;
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    const uint32_t id0 = tc::idesc_mxf4(128, a.Bt, 0), id2 = tc::idesc_mxf4(128, a.Bt, 2);
    const uint32_t hi = tc::desc_hi(1024, tc::kLayoutSw128);
    const uint32_t sf_step = sf_cols(a.groups), sfb_step = 4 * a.groups;
    int s = 0, li = 0;
    uint32_t ph = 0;
    bool go = !kFuse || wait(&aux->x_full, 0);
    for (int item = cid; item < n_items; item += n_cl, ++li) {
      const int acc = li & 1;
      if (li >= 2) go = go && wait(&aux->acc_empty[acc], ((li - 2) >> 1) & 1);
      tc::fence_after_sync();
      const uint32_t d = tmem + uint32_t(kMaxBt) * acc;
      for (int kb = kb0; kb < kb1; ++kb) {
        const uint32_t st = sbase + s * a.stage_bytes;
        const uint32_t sfa = tmem + kColSf + sf_step * s, sfb = sfa + 8;
        const uint32_t xt = kFuse ? sbase + a.x_off + (kb - kb0) * x_tile : st + kWBytes;
        const uint32_t a_lo = tc::desc_lo(st, 16), b_lo = tc::desc_lo(xt, 16);
        go = go && wait(&aux->full[s], ph) && wait(&aux->sf_full[s], ph);
        tc::fence_after_sync();
        if (tc::elect_one() && go) {
#pragma unroll
          for (int ks = 0; ks < KBW / 64; ++ks)
            tc::mma_mxf4(d, tc::desc_pack(a_lo + ks * 2, hi), tc::desc_pack(b_lo + ks * 2, hi), (ks & 1) ? id2 : id0,
                         sfa + 4 * (ks >> 1), sfb + sfb_step * (ks >> 1), (kb > kb0 || ks) ? 1u : 0u);
          tc::mma_commit(smem_u32(&aux->empty[s]));
        }
        __syncwarp();
        if (++s == NS) {
          s = 0;
          ph ^= 1;
        }
      }
      if (tc::elect_one() && go) tc::mma_commit(smem_u32(&aux->acc_full[acc]));
      __syncwarp();
    }
  } else if (warp == 6) {
    // ---------------------------------------------------------------- scales
    // A stage's columns are free once its MMAs have completed, which is when
    // the producer refills the stage: the wait for `full` covers both.
    const uint32_t hi = tc::desc_hi(128, tc::kLayoutNone);
    const uint32_t sf_step = sf_cols(a.groups);
    int s = 0;
    uint32_t ph = 0;
    bool go = !kFuse || wait(&aux->x_full, 0);
    for (int item = cid; item < n_items; item += n_cl) {
      for (int kb = kb0; kb < kb1; ++kb) {
        const uint32_t st = sbase + s * a.stage_bytes;
        const uint32_t sfa = tmem + kColSf + sf_step * s;
        const uint32_t xt = kFuse ? sbase + a.x_off + (kb - kb0) * x_tile : st + kWBytes;
        const uint32_t w_lo = tc::desc_lo(st + kCodeBytes, 16), x_lo = tc::desc_lo(xt + x_bytes, 16);
        go = go && wait(&aux->full[s], ph);
        tc::fence_after_sync();
        if (tc::elect_one() && go) {
          tc::cp_scales(sfa, tc::desc_pack(w_lo, hi));
          tc::cp_scales(sfa + 4, tc::desc_pack(w_lo + 32, hi));
          if (a.groups == 1) {
            tc::cp_scales(sfa + 8, tc::desc_pack(x_lo, hi));
            tc::cp_scales(sfa + 12, tc::desc_pack(x_lo + 32, hi));
          } else {
            tc::cp_scales(sfa + 8, tc::desc_pack(x_lo, hi));
            tc::cp_scales(sfa + 12, tc::desc_pack(x_lo + 64, hi));
            tc::cp_scales(sfa + 16, tc::desc_pack(x_lo + 32, hi));
            tc::cp_scales(sfa + 20, tc::desc_pack(x_lo + 96, hi));
          }
          tc::mma_commit(smem_u32(&aux->sf_full[s]));
        }
        __syncwarp();
        if (++s == NS) {
          s = 0;
          ph ^= 1;
        }
      }
    }
  }

  const bool epilogue = warp >= 2 && warp <= 5;
  const int quarter = warp & 3;        // TMEM lanes [32 quarter, 32 quarter + 32)
  const int nr = quarter * 32 + lane;  // this thread's row of the weight tile
  const uint32_t trow = tmem + ((uint32_t)(quarter * 32) << 16);
  uint8_t* stage = smem + a.out_off;
  const bool lead = tid == 64;
  bool ok = true;  // given up: through the same barriers, without the stores
  if (epilogue) {
    // ---------------------------------------------------------------- epilogue (warps 2-5)
    if (lead && a.tma_store) tma::prefetch_map(&tm_y);
    if constexpr (kFuse) {
      uint8_t* xs = smem + a.x_off;
      if (a.x_type == DSA_BF16)
        fill_x<__nv_bfloat16>(a, xs, x_tile, kb0, kb1, warp - 2, lane);
      else if (a.x_type == DSA_FP16)
        fill_x<__half>(a, xs, x_tile, kb0, kb1, warp - 2, lane);
      else
        fill_x<float>(a, xs, x_tile, kb0, kb1, warp - 2, lane);
      tc::fence_proxy_async();  // the tensor cores read it
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(smem_u32(&aux->x_full));
    }
    if (C == 1) {
      int li = 0;
      for (int item = cid; item < n_items; item += n_cl, ++li) {
        const int acc = li & 1;
        const int t = item / a.m_tiles, mt = item - t * a.m_tiles;
        const int64_t b0 = int64_t(mt) * a.Bt;
        const int rows = int(min(int64_t(a.Bt), a.B - b0));
        if (a.tma_store && li > 0) {  // the tile before has left the staging buffer
          if (lead) lin::bulk_wait_read();
          tc::named_bar_sync(1, 128);
        }
        ok = ok && wait(&aux->acc_full[acc], (li >> 1) & 1);
        __syncwarp();
        tc::fence_after_sync();
        // rows past the tile's tokens are staged too (the store leaves them out)
        const uint32_t tacc = trow + uint32_t(kMaxBt) * acc;
        if (!kF32 && a.tma_store) {
          // 16x256b fragments: thread i holds weight rows i / 4 and 8 + i / 4
          // at tokens 2 (i % 4) + {0, 1}; stmatrix.trans turns 8x8 blocks
          // around: four 16-byte pieces of token rows an instruction
          // (element stores of the transposed tile took 200 cycles a row)
          const int blk = lane >> 3, n0 = quarter * 32 + (blk & 1) * 8;
          for (int c0 = 0; c0 < rows; c0 += 32) {
            float v[2][16];
            tc::tmem_ld16x256b_x4(tacc + c0, v[0]);
            tc::tmem_ld16x256b_x4(tacc + (16u << 16) + c0, v[1]);
            tc::tmem_wait_ld();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
              for (int r = 0; r < 4; r += 2) {
                const uint32_t at = smem_u32(stage_at<false>(stage, a.half_bytes, c0 + 8 * (r + (blk >> 1)) + (lane & 7),
                                                             n0 + 16 * h));
                const float* p = v[h] + 4 * r;
                asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(at),
                             "r"(pack_bf16x2(p[0], p[1])), "r"(pack_bf16x2(p[2], p[3])), "r"(pack_bf16x2(p[4], p[5])),
                             "r"(pack_bf16x2(p[6], p[7]))
                             : "memory");
              }
            }
          }
        } else {
          for (int c0 = 0; c0 < rows; c0 += 32) {
            float v[32];
            tc::tmem_ld32(tacc + c0, v);
            tc::tmem_wait_ld();
            if (a.tma_store) {
#pragma unroll
              for (int i = 0; i < 32; ++i) *stage_at<kF32>(stage, a.half_bytes, c0 + i, nr) = to_out<kF32>(v[i]);
            } else if (ok) {
              store_rows<kF32, 32>(a, b0 + c0, rows - c0, t * TILE_N + nr, v);
            }
          }
        }
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(smem_u32(&aux->acc_empty[acc]));
        if (a.tma_store) {
          tc::fence_proxy_async();
          tc::named_bar_sync(1, 128);
          if (lead && !*static_cast<volatile int*>(&aux->abort))
            store_tile<kF32>(&tm_y, smem_u32(stage), a.half_bytes, t, int(b0), a.N);
        }
      }
    } else {
      ok = __all_sync(0xffffffffu, wait(&aux->acc_full[0], 0)) != 0;
      tc::fence_after_sync();
    }
  }
  if (C > 1) {
    // one item a cluster; every CTA's products are done once all have arrived
    lin::cluster_arrive();
    lin::cluster_wait();
  }
  if (epilogue) {
    if (C > 1) {
      const int t = cid / a.m_tiles, mt = cid - t * a.m_tiles;
      const int64_t b0 = int64_t(mt) * a.Bt;
      const int rows = int(min(int64_t(a.Bt), a.B - b0));
      const int R = a.rows_per, r0 = rank * R, own = max(0, min(rows, r0 + R) - r0);
      float* part = reinterpret_cast<float*>(smem + a.part_off);
      const float* recv = reinterpret_cast<const float*>(smem + a.recv_off);
      if (ok) {
        for (int c0 = 0; c0 < rows; c0 += 32) {
          float v[32];
          tc::tmem_ld32(trow + c0, v);
          tc::tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) part[(c0 + i) * TILE_N + nr] = v[i];  // (room for whole groups of 32)
        }
      } else {
        poison(part + nr, rows, &aux->drained, a.status);
      }
      tc::fence_proxy_async();  // the copy engine reads the partial
      tc::named_bar_sync(1, 128);
      if (lead) {
        tma::mbar_arrive_expect_tx(smem_u32(&aux->ready), uint32_t(C * own) * TILE_N * 4u);
        for (int q = 0; q < C; ++q) {
          const int n = min(R, rows - q * R);
          if (n <= 0) break;
          lin::bulk_to_peer(lin::mapa(smem_u32(recv) + uint32_t(rank * R) * TILE_N * 4u, q),
                            smem_u32(part) + uint32_t(q * R) * TILE_N * 4u, uint32_t(n) * TILE_N * 4u,
                            lin::mapa(smem_u32(&aux->ready), q));
        }
      }
      // every CTA sends, so all copies come: they land before this one leaves
      if (!lin::mbar_wait_cluster(smem_u32(&aux->ready), 0, a.status, a.wait_limit))
        ok = lin::mbar_wait_cluster(smem_u32(&aux->ready), 0, a.status, tc::kWaitCycles) && ok;
      for (int l0 = 0; l0 < own; l0 += 8) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.f;
        for (int q = 0; q < C; ++q) {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] += recv[(q * R + min(l0 + j, R - 1)) * TILE_N + nr];
        }
        if (a.tma_store) {
#pragma unroll
          for (int j = 0; j < 8; ++j) *stage_at<kF32>(stage, a.half_bytes, l0 + j, nr) = to_out<kF32>(v[j]);
        } else if (ok) {
          store_rows<kF32, 8>(a, b0 + r0 + l0, own - l0, t * TILE_N + nr, v);
        }
      }
      if (a.tma_store && own > 0) {
        tc::fence_proxy_async();
        tc::named_bar_sync(1, 128);
        if (lead && ok) store_tile<kF32>(&tm_y, smem_u32(stage), a.half_bytes, t, int(b0) + r0, a.N);
      }
    }
    if (lead) lin::bulk_wait_read();  // the tiles have left shared memory
  } else if (C > 1 && aux->abort) {
    drain(aux, NS, a.status);
  }
  tc::fence_before_sync();
  __syncthreads();
  if (C == 1 && (warp < 2 || warp > 5) && aux->abort) drain(aux, NS, a.status);
  if (C > 1) {  // no CTA leaves while a peer may still touch its shared memory
    lin::cluster_arrive();
    lin::cluster_wait();
  }
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, kTmemCols);
  }
}

// X [B, K] -> its tiles.  A warp takes 2 kQuantUnroll k-blocks of one token,
// a half warp each.
constexpr int kQuantThreads = 256;
constexpr int kQuantUnroll = 2;
template <typename T>
__global__ void __launch_bounds__(kQuantThreads) quant_x_kernel(const T* __restrict__ x, int64_t ld_x,
                                                                uint8_t* __restrict__ tiles, int B, int K, int Bt,
                                                                int groups, int nkb) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int runs = (nkb + 2 * kQuantUnroll - 1) / (2 * kQuantUnroll);  // of a token
  const int64_t total = int64_t(B) * runs, step = int64_t(gridDim.x) * (kQuantThreads / 32);
  for (int64_t w = int64_t(blockIdx.x) * (kQuantThreads / 32) + (threadIdx.x >> 5); w < total; w += step) {
    // (a 64-bit division was a quarter of the instructions)
    const int b = total < (int64_t(1) << 32) ? int(uint32_t(w) / uint32_t(runs)) : int(w / runs);
    const int kb0 = int(w - int64_t(b) * runs) * 2 * kQuantUnroll + (lane >> 4);
    KBlock<T> v[kQuantUnroll];
#pragma unroll
    for (int u = 0; u < kQuantUnroll; ++u)
      v[u] = load_kblock(x + b * ld_x, kb0 + 2 * u, K, lane, kb0 + 2 * u < nkb);
    const int mt = int(uint32_t(b) / uint32_t(Bt)), r = b - mt * Bt;
    const int tile_bytes = Bt * (KBW / 2) + groups * kSfBytes;
    uint8_t* tile = tiles + (int64_t(mt) * nkb + kb0) * tile_bytes;
#pragma unroll
    for (int u = 0; u < kQuantUnroll; ++u)
      put_kblock<T>(tile + 2 * u * tile_bytes, v[u], Bt, r, lane, kb0 + 2 * u < nkb);
  }
}

// codes [N, K/2], scales [N, K/32] row-major -> the weight tiles, 16 B a thread
__global__ void pack_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                            uint8_t* __restrict__ out, int N, int K, int nkb, int64_t chunks) {
  constexpr int kChunks = kWBytes / 16;  // of a tile
  for (int64_t id = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; id < chunks; id += int64_t(gridDim.x) * blockDim.x) {
    const int64_t tile = id / kChunks;
    const int within = int(id - tile * kChunks);
    const int kb = int(tile % nkb), t = int(tile / nkb);
    uint4 v = make_uint4(0, 0, 0, 0);
    uint8_t* dst = out + tile * kWBytes;
    if (within < kCodeBytes / 16) {
      const int r = within >> 3, c = within & 7;
      const int n = t * TILE_N + r, k = kb * KBW + c * 32;
      if (n < N && k < K) v = *reinterpret_cast<const uint4*>(codes + int64_t(n) * (K / 2) + k / 2);
      dst += r * 128 + ((c ^ (r & 7)) << 4);
    } else {
      // 16 B of scales: rows r, r + 32, r + 64, r + 96, four scales each
      const int s = within - kCodeBytes / 16, half = s >> 5, r = s & 31;
      uint8_t* b = reinterpret_cast<uint8_t*>(&v);
      for (int q = 0; q < 4; ++q) {
        const int n = t * TILE_N + q * 32 + r;
        for (int j = 0; j < 4; ++j) {
          const int i = kb * kSfPerKb + half * 4 + j;
          if (n < N && i < K / mx::kBlock) b[q * 4 + j] = scales[int64_t(n) * (K / mx::kBlock) + i];
        }
      }
      dst += kCodeBytes + s * 16;
    }
    *reinterpret_cast<uint4*>(dst) = v;
  }
}

// Clusters of C CTAs that can be resident at once (one CTA per SM), C = 1 ..
// kMaxSplit, for the current device; NULL without one.  Filled at its first
// call on a device, which also raises the kernels' shared-memory limit.
static const int* cluster_table() {
  static int table[64][kMaxSplit + 1];
  static std::once_flag once[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    cudaGetLastError();
    return nullptr;
  }
  std::call_once(once[dev], [dev] {
    int* n = table[dev];
    for (auto k : {linear_mxfp4_kernel<false, false>, linear_mxfp4_kernel<true, false>, linear_mxfp4_kernel<false, true>,
                   linear_mxfp4_kernel<true, true>}) {
      if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes) != cudaSuccess ||
          cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
        cudaGetLastError();
        return;
      }
    }
    n[1] = num_sms();
    for (int C = 2; C <= kMaxSplit; ++C) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(C);
      cfg.blockDim = dim3(THREADS);
      cfg.dynamicSmemBytes = kSmemBytes;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = C;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&n[C], linear_mxfp4_kernel<false, false>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        n[C] = 0;
      }
    }
  });
  return table[dev][1] > 0 ? table[dev] : nullptr;
}

struct Plan {
  int Bt, m_tiles, groups, split;
  int fuse;  // k-blocks of X that a CTA quantises itself (0: X is quantised by its own launch)
};

// shared memory of a plan: the ring's stages (0: it does not fit) and offsets
static int lay_out(const Plan& p, int B, int es, bool tma_store, Args* a) {
  const int tokens = std::min(B, p.Bt);
  const int R = (tokens + p.split - 1) / p.split;
  // whole groups of rows as the epilogue writes them: 32, a split's owner 8
  const int out_rows = p.split > 1 ? (R + 7) / 8 * 8 : (p.Bt + 31) / 32 * 32;
  const uint32_t x_tile = uint32_t(p.Bt * (KBW / 2) + p.groups * kSfBytes);
  const uint32_t stage = kWBytes + (p.fuse ? 0u : x_tile), x_region = uint32_t(p.fuse) * x_tile;
  const uint32_t out_bytes = tma_store ? (uint32_t(out_rows) * TILE_N * es + 1023u) & ~1023u : 0u;
  const uint32_t part = p.split > 1 ? uint32_t((tokens + 31) / 32 * 32) * TILE_N * 4 : 0u;
  const uint32_t recv = p.split > 1 ? uint32_t(p.split * R) * TILE_N * 4 : 0u;
  const uint32_t room = kSmemBytes - 1024 - kAuxBytes;
  if (out_bytes + x_region >= room || part + recv + out_bytes > room) return 0;
  const int stages = std::min<int>(max_stages(p.groups), (room - out_bytes - x_region) / stage);
  if (stages < 2) return 0;
  // the partials take the ring's place; the staged tile starts on 1024 B
  const uint32_t ring = (std::max(stages * stage + x_region, part + recv) + 1023u) & ~1023u;
  if (ring + out_bytes > room) return 0;
  if (a) {
    a->n_stages = stages;
    a->stage_bytes = stage;
    a->rows_per = R;
    a->half_bytes = uint32_t(out_rows) * 128;
    a->x_off = stages * stage;
    a->part_off = 0;
    a->recv_off = part;
    a->out_off = ring;
    a->aux_off = ring + out_bytes;
  }
  return stages;
}

// Tokens an item and CTAs an item: the pair with the lowest estimate of the
// busiest CTA's cycles.  A k-block takes its issuers ~550 cycles and its bytes
// ~70 a cycle into the SM (at 192 tokens 630 measured); an item a fixed ~1.5K
// cycles and its share of the epilogue; a split its cluster's start and
// barriers, the exchange of its partial and the sum of C of them.  Half of the
// time that all bytes would take at 50 a cycle and SM breaks ties towards
// fewer re-reads.  Measured over 18 shapes x 60 pairs the pick is within 7 % of the
// best; splitting pays below ~64 tokens (64 x 4096 x 8192: 10.6 us with C = 4, 12.7
// unsplit; 128 x 4096 x 8192: 14.6 with C = 4, 13.7 unsplit).
static Plan pick_plan(int B, int N, int nkb) {
  static const int kNone[kMaxSplit + 1] = {0, 148};  // no device: unsplit
  const int* clusters = cluster_table();
  if (!clusters) clusters = kNone;
  // a call asks twice (its workspace's size, then the launch)
  struct Asked {
    const int* clusters;
    int B, N, nkb;
    Plan plan;
  };
  static thread_local Asked last{};
  if (last.clusters == clusters && last.B == B && last.N == N && last.nkb == nkb) return last.plan;
  const int n_tiles = (N + TILE_N - 1) / TILE_N;
  Plan best{};
  double best_cost = 0;
  for (int want : {32, 48, 64, 96, 128, 160, 192}) {
    const int m_tiles = (B + want - 1) / want;
    const int Bt = std::max(32, ((B + m_tiles - 1) / m_tiles + 15) / 16 * 16);
    const int64_t items = int64_t(n_tiles) * m_tiles;
    const double tokens = std::min(B, Bt);
    const double kb_bytes = kWBytes + Bt * 136.0, kb_cost = std::max(550.0, kb_bytes / 70.0);
    const double all_bytes = items * double(nkb) * kb_bytes / (50.0 * clusters[1]);
    for (int C = 1; C <= std::min(kMaxSplit, nkb); ++C) {
      if (C > 1 && items > clusters[C]) continue;
      Plan p{Bt, m_tiles, (Bt + 127) / 128, C, 0};
      if (!lay_out(p, B, 4, true, nullptr)) continue;
      const int64_t waves = C > 1 ? 1 : (items + clusters[1] - 1) / clusters[1];
      const double cost = waves * ((nkb + C - 1) / C * kb_cost + 1500) + Bt * 8.0 + 0.5 * all_bytes +
                          (C > 1 ? 3000 + (40.0 + 0.4 * tokens) * tokens + 250.0 * C : 0);
      if (best.Bt == 0 || cost < best_cost) {
        best_cost = cost;
        best = p;
      }
    }
  }
  // Quantising X in the product saves a launch and X's way through memory and
  // costs each CTA its share of X on four warps.  Measured, fused against two
  // launches: 1 x 1024 x 4096 (2 units a CTA) 4.9 / 5.6 us, 8 x 1024 x 4096
  // (16) 5.45 / 6.1, 16 x 1024 x 4096 (32) 6.3 / 6.3, 12 x 32768 x 1024 (48) 7.0 /
  // 6.7, 24 x 1024 x 4096 (48) 7.0 / 6.45, 16 x 32768 x 1024 (64) 7.6 / 6.7.
  const int share = (nkb + best.split - 1) / best.split;
  if (best.m_tiles == 1 && int64_t(share) * B <= kFuseUnits) {
    Plan f = best;
    f.fuse = share;
    if (lay_out(f, B, 4, true, nullptr)) best = f;
  }
  last = {clusters, B, N, nkb, best};
  return best;
}

static size_t x_bytes_for(const Plan& p, int nkb) {
  if (p.fuse) return 0;
  return size_t(p.m_tiles) * nkb * (p.Bt * (KBW / 2) + p.groups * kSfBytes);
}
static int n_kblocks(int K) { return (K + KBW - 1) / KBW; }
static bool good_sizes(int64_t B, int64_t N, int64_t K) {
  return B >= 0 && B <= (1 << 24) && N > 0 && N <= (1 << 24) && K > 0 && K <= (1 << 24) && K % mx::kBlock == 0;
}

}  // namespace lmx
}  // namespace dsa

using namespace dsa;

extern "C" size_t dsa_linear_mxfp4_packed_bytes(int N, int K) {
  if (!lmx::good_sizes(0, N, K)) return 0;
  return size_t((N + lmx::TILE_N - 1) / lmx::TILE_N) * lmx::n_kblocks(K) * lmx::kWBytes;
}

extern "C" int dsa_linear_mxfp4_pack(const uint8_t* codes, const uint8_t* scales, int N, int K, void* packed,
                                     size_t packed_bytes, dsa_stream_t stream) {
  clear_error();
  DSA_CHECK_ARG(codes && scales && packed, "linear_mxfp4_pack: null codes/scales/packed");
  DSA_CHECK_ARG(lmx::good_sizes(0, N, K), "linear_mxfp4_pack: bad N/K (K a multiple of 32, at most 2^24)");
  DSA_CHECK_ARG(aligned(codes, 16) && aligned(packed, 16), "linear_mxfp4_pack: codes/packed must be 16-byte aligned");
  const size_t need = dsa_linear_mxfp4_packed_bytes(N, K);
  DSA_CHECK_ARG(packed_bytes >= need, "linear_mxfp4_pack: packed buffer %zu bytes < %zu", packed_bytes, need);
  const int64_t chunks = int64_t(need / 16);
  const int grid = int(std::min<int64_t>((chunks + 255) / 256, int64_t(num_sms()) * 16));
  lmx::pack_kernel<<<grid, 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      codes, scales, static_cast<uint8_t*>(packed), N, K, lmx::n_kblocks(K), chunks);
  DSA_CHECK_LAUNCH("linear_mxfp4_pack");
  return DSA_OK;
}

extern "C" size_t dsa_linear_mxfp4_workspace_size(int B, int N, int K) {
  if (!lmx::good_sizes(B, N, K) || B == 0) return 0;
  const int nkb = lmx::n_kblocks(K);
  const lmx::Plan p = lmx::pick_plan(B, N, nkb);
  return lmx::x_bytes_for(p, nkb);
}

extern "C" int dsa_linear_mxfp4(const void* x, int x_type, int64_t ld_x, const void* w_packed, void* y, int64_t ld_y,
                                int B, int N, int K, int out_f32, void* workspace, size_t workspace_bytes,
                                int32_t* status, dsa_stream_t stream) {
  clear_error();
  DSA_CHECK_ARG(x && w_packed && y, "linear_mxfp4: null x/w/y");
  DSA_CHECK_ARG(x_type == DSA_BF16 || x_type == DSA_FP16 || x_type == DSA_FP32, "linear_mxfp4: unknown x_type %d",
                x_type);
  DSA_CHECK_ARG(lmx::good_sizes(B, N, K), "linear_mxfp4: bad B/N/K (K a multiple of 32, each at most 2^24)");
  const int xs = x_type == DSA_FP32 ? 4 : 2, es = out_f32 ? 4 : 2;
  DSA_CHECK_ARG(aligned(x, 16) && aligned(w_packed, 16) && (B <= 1 || (ld_x >= K && ld_x * xs % 16 == 0)),
                "linear_mxfp4: x needs 16-byte alignment and a row stride >= K, a multiple of 16 bytes");
  DSA_CHECK_ARG((B <= 1 || ld_y >= N) && aligned(y, es), "linear_mxfp4: ld_y < N, or y not aligned to its type");
  if (B == 0) return DSA_OK;
  const int nkb = lmx::n_kblocks(K);
  const lmx::Plan p = lmx::pick_plan(B, N, nkb);
  if (p.Bt == 0) {
    set_error("linear_mxfp4: no launch configuration fits");
    return DSA_ERR_CUDA;
  }
  DSA_CHECK_ARG(int64_t((N + lmx::TILE_N - 1) / lmx::TILE_N) * p.m_tiles <= INT32_MAX, "linear_mxfp4: B*N is too large");
  const size_t need = lmx::x_bytes_for(p, nkb);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16))) {
    set_error("linear_mxfp4: needs %zu bytes of 16-byte aligned workspace (got %zu)", need, workspace_bytes);
    return DSA_ERR_WORKSPACE;
  }
  uint8_t* tiles = static_cast<uint8_t*>(workspace);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);

  lmx::Args a{};
  a.w = static_cast<const uint8_t*>(w_packed);
  a.x = p.fuse ? static_cast<const uint8_t*>(x) : tiles;
  a.ld_x = ld_x;
  a.x_type = x_type;
  a.K = K;
  a.y = y;
  a.ld_y = ld_y;
  a.B = B;
  a.Bt = p.Bt;
  a.groups = p.groups;
  a.N = N;
  a.nkb = nkb;
  a.n_tiles = (N + lmx::TILE_N - 1) / lmx::TILE_N;
  a.m_tiles = p.m_tiles;
  a.split = p.split;
  a.tma_store = aligned(y, 16) && (B == 1 || ld_y * es % 16 == 0) && int64_t(N) * es % 16 == 0 ? 1 : 0;
  // a split's last owner may hold fewer rows than its box: below the last
  // token tile the box would reach into the next one
  if (p.split > 1 && p.m_tiles > 1 && p.Bt % p.split != 0) a.tma_store = 0;
  a.status = status;
  a.wait_limit = wait_limit_cycles();
  if (!lmx::cluster_table() || !lmx::lay_out(p, B, es, a.tma_store, &a)) {
    set_error("linear_mxfp4: no launch configuration fits");
    return DSA_ERR_CUDA;
  }
  CUtensorMap tm_y;
  memset(&tm_y, 0, sizeof(tm_y));
  if (a.tma_store) {
    tma::EncodeTiledFn fn = tma::encode_fn();
    const cuuint64_t dims[2] = {uint64_t(N), uint64_t(B)};
    const cuuint64_t strides[1] = {uint64_t(B == 1 ? N : ld_y) * es};
    const cuuint32_t box[2] = {uint32_t(out_f32 ? lmx::TILE_N : 64), uint32_t(p.split > 1 ? a.rows_per : p.Bt)};
    const cuuint32_t estr[2] = {1, 1};
    if (!fn || fn(&tm_y, out_f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, y, dims,
                  strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  out_f32 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
      set_error("linear_mxfp4: cuTensorMapEncodeTiled (Y) failed");
      return DSA_ERR_CUDA;
    }
  }
  if (!p.fuse) {
    const int64_t q_warps = int64_t(B) * ((nkb + 2 * lmx::kQuantUnroll - 1) / (2 * lmx::kQuantUnroll));
    const int per = lmx::kQuantThreads / 32;
    const dim3 qgrid(unsigned(std::min<int64_t>((q_warps + per - 1) / per, int64_t(num_sms()) * 32)));
    auto quant = [&](auto* ptr) {
      using T = std::remove_pointer_t<decltype(ptr)>;
      launch_pdl(lmx::quant_x_kernel<T>, qgrid, dim3(lmx::kQuantThreads), 0, st, static_cast<const T*>(x), ld_x,
                 tiles, B, K, p.Bt, p.groups, nkb);
    };
    if (x_type == DSA_BF16)
      quant(static_cast<__nv_bfloat16*>(nullptr));
    else if (x_type == DSA_FP16)
      quant(static_cast<__half*>(nullptr));
    else
      quant(static_cast<float*>(nullptr));
    DSA_CHECK_LAUNCH("linear_mxfp4 (quantisation)");
  }
  const int64_t items = int64_t(a.n_tiles) * a.m_tiles;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(p.split > 1 ? items * p.split : std::min<int64_t>(items, num_sms())));
  cfg.blockDim = dim3(lmx::THREADS);
  cfg.dynamicSmemBytes = lmx::kSmemBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.split;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.split > 1 ? 2 : 1;
  auto kernel = p.fuse ? (out_f32 ? lmx::linear_mxfp4_kernel<true, true> : lmx::linear_mxfp4_kernel<false, true>)
                       : (out_f32 ? lmx::linear_mxfp4_kernel<true, false> : lmx::linear_mxfp4_kernel<false, false>);
  cudaLaunchKernelEx(&cfg, kernel, a, tm_y);
  DSA_CHECK_LAUNCH("linear_mxfp4");
  return DSA_OK;
}
